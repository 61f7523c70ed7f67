// Decode attention over a paged cache: a few new rows of each sequence, split over the sequences' lengths and joined.
//
// For row t of a sequence of L keys with n rows: s_j = scale q_t . k_j over keys j <= L - n + t (causal) or all L,
// out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m). Splits of the keys keep (m, l, acc) and are joined as
// M = max m, out = sum e^(m - M) acc / sum e^(m - M) l.
//
// What bounds it. Long batches: each key and value is read once from HBM, since the heads of a group and the sequence's rows share
// one pass (64 sequences of 0.1k-8k keys, Llama-3-8B heads, f16: 1.09 GB in 182 us, 6.0 TB/s). Short calls: a few dependent round
// trips (513 keys, Qwen2.5-0.5B heads, 6.3 us, of which an empty launch is 2; 8192 keys, Llama-3-8B heads, 11.3 us: 1 to find the
// chunk, 5 to its keys, 1 to join the waves, 1.5 to publish and count, 2 for the last one's join).
//
//   * The lengths are in device memory, so that a captured launch replays while sequences grow: the grid is fixed by the host
//     and every workgroup works out its own part from the lengths, 64 sequences a step. Small launches take chunks, one
//     (sequence, kv head, tile of query rows, chunk of keys) for a workgroup; large ones take ranges: an equal share of the list of
//     all sequences' keys for each workgroup that the chip holds, walked over the sequences in it without a break.
//   * Each wave walks every NW-th block of 32 keys with the next blocks in flight in registers; keys and values reach the operand
//     layouts of v_mfma_f32_16x16x32 through LDS, values through its transposing read, and the probabilities never leave registers.
//   * A page holds at least 16 keys, so the 16-key halves of a block each lie in one page: two page numbers per block, read one
//     block ahead of the keys they place.
//   * Parts of a sequence publish their partials with device-scope stores and count themselves in; the last one of a tile joins them
//     in order (the result does not depend on which was last) and resets the counter.
#include "mx_paged.hpp"

namespace mx {

namespace {

constexpr int kBlock = kPagedDecodeBlock;

typedef short short4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ u32x2 load8_dev(__amdgpu_buffer_rsrc_t r, int byte_off) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(r, byte_off, 0, kCpolSc1));
}

// Quanta of QK keys of a sequence. One at least: an empty sequence's rows are written too. whole: sequences are not split.
template <int QK>
__device__ __forceinline__ int quanta_of(const PagedAttnParams & p, int len) {
    return !p.whole && length_ok(p.c, len) ? max(1, (len + QK - 1) / QK) : 1;
}

// ---- a workgroup's part of the launch, the same in all its waves ----

// Chunks: one (sequence, chunk of its keys) for a workgroup.
struct Chunk {
    int32_t b;        // sequence, -1: nothing
    int32_t len;      // its kv_len as it is
    int32_t i, n;     // chunk and chunks of it
    int32_t keys;     // keys of a chunk (the last takes what is left)
    int32_t ordinal;  // sequences of several chunks before it
    int32_t slot;     // chunks of those
};

// The j-th chunk of the launch, planned from the lengths of all sequences (64 a step). Where none is longer than p.whole_keys keys
// each is one chunk: joining costs more than the walk saves. Else the chunks, of the shorter sequences too, are the shortest that
// the launch has workgroups for.
template <int QK>
__device__ __forceinline__ Chunk find_chunk(const PagedAttnParams & p, int j, int lane) {
    const int n_seq = p.c.n_seq;
    const int len0 = p.c.kv_len[min(lane, n_seq - 1)];
    auto len_of = [&](int base) { return base == 0 ? len0 : p.c.kv_len[min(base + lane, n_seq - 1)]; };
    auto quanta = [&](int base, int len) { return base + lane < n_seq ? quanta_of<QK>(p, len) : 0; };
    int longest = 0;
    float sum = 0.f;  // of quanta: only the plan depends on it
    for (int base = 0; base < n_seq; base += kWave) {
        const int len = len_of(base);
        if (length_ok(p.c, len)) longest = max(longest, len);
        sum += (float)quanta(base, len);
    }
    longest = wave_imax(longest);
    const int most = quanta_of<QK>(p, longest);
    sum = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(wave_sum(sum))));
    auto count = [&](int c) {
        int r = 0;
        for (int base = 0; base < n_seq; base += kWave) r += (uint32_t)(quanta(base, len_of(base)) + c - 1) / (uint32_t)c;
        return wave_isum(r);
    };
    int c = most;
    if (longest > p.whole_keys) {
        const int share = __builtin_amdgcn_readfirstlane((int)fminf(ceilf(sum / (float)p.ranges), (float)most));
        c = max((most + kPagedMaxParts - 1) / kPagedMaxParts, share);
        for (int i = 0; c < most && count(c) > p.ranges; i++) c = i < 16 ? min(c + max(1, c / 8), most) : most;
    }
    Chunk x{-1, 0, 0, 1, c * QK, 0, 0};
    int before = 0;
    for (int base = 0; base < n_seq; base += kWave) {
        const int len = len_of(base), n = (uint32_t)(quanta(base, len) + c - 1) / (uint32_t)c;
        const int upto = before + wave_iscan(n);
        const uint64_t many = __builtin_amdgcn_ballot_w64(n > 1);
        const uint64_t past = __builtin_amdgcn_ballot_w64(upto > j);
        if (past) {
            const int l = __builtin_ctzll(past);
            x.b = base + l;
            x.n = __builtin_amdgcn_readlane(n, l);
            x.len = __builtin_amdgcn_readlane(len, l);
            const int first = __builtin_amdgcn_readlane(upto, l) - x.n;
            x.i = j - first;
            x.ordinal += __builtin_popcountll(many & ((1ull << l) - 1));
            x.slot = first - (x.b - x.ordinal);  // the other sequences before it have one chunk each
            return x;
        }
        before = __builtin_amdgcn_readlane(upto, 63);
        x.ordinal += __builtin_popcountll(many);
    }
    return x;
}

// Ranges: quanta lo .. hi - 1 of the list of all sequences' quanta, one sequence behind the other, for a workgroup, and where
// they start: sequence b, whose first quantum is number at. Each range takes `share` quanta.
struct Range {
    int32_t lo, hi, share;
    int32_t b, at;
};

// Range r: every wave sums all lengths, each lane those of per_lane sequences in a row, and looks for the sequence that holds its
// first quantum. lens: the lengths of the 64 sequences from lens0 on, that one among them.
template <int QK>
__device__ __forceinline__ Range find_range(const PagedAttnParams & p, int r, int lane, int & lens, int & lens0) {
    const int n_seq = p.c.n_seq, per_lane = (n_seq + kWave - 1) / kWave;
    lens = p.c.kv_len[min(lane, n_seq - 1)];
    lens0 = 0;
    int mine = 0, most = 0;
    if (per_lane == 1) {
        mine = most = lane < n_seq ? quanta_of<QK>(p, lens) : 0;
    } else {
        constexpr int kAtOnce = 8;
        for (int i0 = 0; i0 < per_lane; i0 += kAtOnce) {
            int len[kAtOnce];
#pragma unroll
            for (int e = 0; e < kAtOnce; e++) len[e] = p.c.kv_len[min(lane * per_lane + i0 + e, n_seq - 1)];
#pragma unroll
            for (int e = 0; e < kAtOnce; e++) {
                const bool in = i0 + e < per_lane && lane * per_lane + i0 + e < n_seq;
                const int n = in ? quanta_of<QK>(p, len[e]) : 0;
                mine += n;
                most = max(most, n);
            }
        }
    }
    const int sum = wave_isum(mine);
    most = wave_imax(most);
    // an equal share each, and no more parts of a sequence than the merge takes (a part may start within a range: one more)
    Range x;
    x.share = max((sum + p.ranges - 1) / p.ranges, (most + kPagedMaxParts - 2) / (kPagedMaxParts - 1));
    const int64_t lo = (int64_t)r * x.share;
    x.lo = (int)min(lo, (int64_t)sum);
    x.hi = (int)min(lo + x.share, (int64_t)sum);
    x.b = -1;
    x.at = 0;
    if (x.lo >= x.hi) return x;
    const int upto = wave_iscan(mine);
    const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > x.lo));  // lo < sum: there is one
    x.b = l * per_lane;
    x.at = __builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(mine, l);
    const int end = min(x.b + per_lane, n_seq);
    while (per_lane > 1) {  // among the lane's sequences
        lens0 = x.b;
        lens = p.c.kv_len[min(lens0 + lane, n_seq - 1)];
        const int n = lens0 + lane < end ? quanta_of<QK>(p, lens) : 0, to = x.at + wave_iscan(n);
        const uint64_t past = __builtin_amdgcn_ballot_w64(to > x.lo);
        if (past) {
            const int i = __builtin_ctzll(past);
            x.b = lens0 + i;
            x.at = __builtin_amdgcn_readlane(to, i) - __builtin_amdgcn_readlane(n, i);
            break;
        }
        x.at = __builtin_amdgcn_readlane(to, 63);
        x.b = min(lens0 + kWave, n_seq - 1);
        if (lens0 + kWave >= end) break;  // only where lengths changed meanwhile
    }
    return x;
}

// A barrier for what the waves exchange through LDS: the loads in flight stay so.
__device__ __forceinline__ void lds_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Keys and values past the caches: they are read once (64 sequences of 0.1k to 8k keys, Llama-3-8B heads, 214 -> 195 us).
__device__ __forceinline__ u32x4 load_kv(const char * a) {
    return __builtin_nontemporal_load((const __attribute__((address_space(1))) u32x4 *)(a));
}

// HD: head_dim. RT: query rows per tile (4, 8, 16 or 32; the matrix products have 16 or 32, the others are zero). T: type of
// pages and query rows. NW: waves. RANGES: a workgroup walks a range of the launch's keys over the sequences in it, else one chunk.
template <int HD, int RT, class T, int NW, bool RANGES>
__global__ __launch_bounds__(NW * kWave) __attribute__((amdgpu_waves_per_eu(HD == 256 || RANGES ? 1 : 2)))
void paged_decode_kernel(PagedAttnParams p) {
    constexpr int QT = RT > 16 ? 2 : 1;  // 16-row product tiles
    constexpr int KS = HD / 32;          // product steps along head_dim
    constexpr int LPR = HD / 8;          // lanes per key row
    constexpr int KPL = kWave / LPR;     // key rows per load
    constexpr int NL = kBlock / KPL;     // loads per lane per block, for each of keys and values
    constexpr int VP = HD + 16;          // LDS row pitch of a block's values (conflict-free transposing reads) ...
    constexpr int KPD = HD + 8;          // ... and keys, which pass through the same LDS first
    constexpr int DT = HD / 16;
    constexpr int kThreads = NW * kWave;
    constexpr int kStep = NW * kBlock;   // keys of a quantum: a block for each wave
    constexpr int PR = HD + 4;           // floats of a partial's row: acc, m, l
    // Blocks of a wave in flight. Chunks are short and few: their walk is one memory round trip per block unless the next blocks
    // are out already, as many as fit the registers (513 keys, Qwen2.5-0.5B heads, 7.3 us with one, 6.4 with three). Ranges keep
    // the memory busy with one, and their registers go to a second workgroup.
    constexpr int D = RANGES || HD == 256 || (HD == 128 && RT == 32) ? 1 : HD == 64 && RT <= 16 ? 3 : 2;
    constexpr int SS = RT * PR;
    constexpr int NQ = RT * HD / 4;      // output quads of the tile
    constexpr int kLds = kBlock * VP * 2 > RT * HD * 4 ? kBlock * VP * 2 : RT * HD * 4;  // bytes of a wave: block, then outputs
    static_assert(16 % KPL == 0, "a load's rows lie in one page");
    __shared__ __attribute__((aligned(16))) char s_buf[NW][kLds];
    __shared__ float s_m[NW][RT], s_l[NW][RT];
    __shared__ int s_last;
    auto s_o = [&](int w) { return reinterpret_cast<float *>(s_buf[w]); };

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
    // kv heads fastest (workgroups are dealt to the 8 XCDs round-robin), the row tiles of one range on one XCD, 8 ids apart:
    // all but the first find its keys in that XCD's L2
    const uint32_t id = blockIdx.x, tiles = p.n_rowtiles;
    const uint32_t grp = id / (8 * tiles) * 8 + id % 8;
    const int rt = id / 8 % tiles, g = grp % p.n_head_kv, r = grp / p.n_head_kv;
    if (r >= p.ranges) return;  // the grid in whole rounds of XCDs
    const int G = p.group, n_q = p.n_q, n_seq = p.c.n_seq;
    const int64_t per_seq = (int64_t)p.n_head_kv * p.n_rowtiles, tile = (int64_t)rt * p.n_head_kv + g;

    const int srow = lane % 16, sgrp = lane / 16;           // score lanes: query row, keys 4 sgrp .. + 4 of a 16-key tile
    const int vslot = lane / LPR, vcol = 8 * (lane % LPR);  // load lanes: key row, first dim
    const int64_t head = (int64_t)g * p.c.head_stride;
    const int shift = p.c.page_shift, page_mask = (1 << shift) - 1;
    const uint32_t kv_stride = (uint32_t)p.c.kv_stride;
    // page numbers of the two halves of the block at key jb, in lanes 0 and 1 (past the table: its last entry; numbers behind the
    // last key are not used)
    auto read_ids = [&](int b, int jb) {
        return p.c.table[b * p.c.table_stride + min((uint32_t)(jb + 16 * (lane & 1)) >> shift, (uint32_t)p.max_pages - 1)];
    };

    // this lane's rows of a product tile: local row, sequence row, head, last visible key
    u32x4 q[QT][KS];
    auto row_ok = [&](int t) { return 16 * t + srow < RT && rt * RT + 16 * t + srow < p.rows; };
    auto load_q = [&](int b) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < QT; t++) {
            const int rr = row_ok(t) ? rt * RT + 16 * t + srow : 0;  // a row past the tile: the problem's first, zeroed
            const uint16_t * qr = p.q + ((int64_t)b * n_q + rr / G) * p.q_stride + (int64_t)(g * G + rr % G) * HD + 8 * sgrp;
#pragma unroll
            for (int ks = 0; ks < KS; ks++) q[t][ks] = load16(qr + 32 * ks);
        }
    };
    // a part of a sequence: its keys up to k1 - 1, for sequence b of L keys (-1: a length that is none); RANGES: its first quantum
    // is number at
    struct Seg {
        int b, at, L, k1;
    };
    Seg seg;
    int key0, ids[D];
    Range x{};
    Chunk ch{};
    int lens = 0, lens0 = 0;  // RANGES: the lengths of 64 sequences from lens0 on
    auto segment = [&](Seg & s, int len) __attribute__((always_inline)) {  // of s.b and s.at; returns its first key
        s.L = length_ok(p.c, len) ? len : -1;
        const int q1 = x.hi - s.at;
        s.k1 = p.whole || q1 >= quanta_of<kStep>(p, s.L) ? max(s.L, 0) : q1 * kStep;
        return max(x.lo - s.at, 0) * kStep;
    };
    auto next_segment = [&](Seg & s) __attribute__((always_inline)) {
        if constexpr (RANGES) {
            s.at += quanta_of<kStep>(p, s.L);
            if (s.at < x.hi) {
                s.b++;
                if ((uint32_t)(s.b - lens0) >= (uint32_t)kWave) {
                    lens0 = s.b;
                    lens = p.c.kv_len[min(lens0 + lane, n_seq - 1)];
                }
                segment(s, __builtin_amdgcn_readlane(lens, s.b - lens0));
                return;
            }
        }
        s.b = -1;
    };
    if constexpr (RANGES) {
        x = find_range<kStep>(p, r, lane, lens, lens0);
        if (x.b < 0) return;  // uniform over the workgroup
        seg.b = x.b;
        seg.at = x.at;
        key0 = segment(seg, __builtin_amdgcn_readlane(lens, x.b - lens0));
    } else {
        if (p.fixed) {
            // the host found room for p.fixed chunks of a quantum for every sequence: the chunk follows from the workgroup's
            // number, and its length and first page numbers are one round trip instead of two
            ch.i = (uint32_t)r / (uint32_t)n_seq;
            ch.b = r - ch.i * n_seq;
#pragma unroll
            for (int i = 0; i < D; i++) ids[i] = read_ids(ch.b, (ch.i + i) * kStep + kBlock * wave);
            ch.len = __builtin_amdgcn_readfirstlane(p.c.kv_len[ch.b]);
            ch.keys = kStep;
            ch.n = min(p.fixed, quanta_of<kStep>(p, ch.len));
            if (ch.len <= p.whole_keys) ch.n = 1;
            if (ch.i >= ch.n) return;
            ch.ordinal = ch.b;
            ch.slot = ch.b * p.fixed;
        } else {
            ch = find_chunk<kStep>(p, r, lane);
            if (ch.b < 0) return;  // uniform over the workgroup
#pragma unroll
            for (int i = 0; i < D; i++) ids[i] = read_ids(ch.b, ch.i * ch.keys + i * kStep + kBlock * wave);
        }
        seg.b = ch.b;
        seg.at = 0;
        seg.L = length_ok(p.c, ch.len) ? ch.len : -1;
        key0 = ch.i * ch.keys;
        seg.k1 = ch.i == ch.n - 1 ? max(seg.L, 0) : key0 + ch.keys;
    }

    // where a block's two halves lie (bytes into the pools), and the last of 16 rows that holds a key
    struct Place {
        int64_t base[2];
        int last[2];
    };
    bool bad_page = false;  // whether a page of the last block placed is none
    auto place = [&](int L, int jb, int ids) __attribute__((always_inline)) {
        Place a;
        bad_page = false;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const bool in = jb + 16 * h < L;  // a half behind the last key repeats the half before it
            int id = __builtin_amdgcn_readlane(ids, in ? h : 0);
            const bool ok = page_ok(p.c, id);
            bad_page |= !ok;
            id = ok ? id : 0;
            const int k16 = jb + (in ? 16 * h : 0);
            a.base[h] = 2 * (head + (int64_t)id * p.c.page_stride + (int64_t)(k16 & page_mask) * p.c.kv_stride);
            a.last[h] = L - 1 - k16;
        }
        return a;
    };
    load_q(seg.b);  // ahead of the keys: a wait for it leaves those in flight
    u32x4 kr[D][NL], vr[D][NL];
    auto load = [&](const uint16_t * pool, const Place & a, u32x4 (&w)[NL]) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < NL; i++) {
            const int h = KPL * i / 16, row = min(KPL * i % 16 + vslot, a.last[h]);
            const char * base = reinterpret_cast<const char *>(pool) + a.base[h];  // the same in every lane
            w[i] = load_kv(base + ((uint32_t)row * kv_stride + vcol) * 2u);
        }
    };
    // RANGES: the wave's blocks over the segments of the range: block `jb` of sequence `jseq` is being computed or in flight, the
    // page numbers of the one behind it (jb_after of sequence `ahead`) are read ahead
    Seg ahead = seg;
    int jb_after = key0 + kBlock * wave, jseq = -1, jb = 0, ids_after = 0;
    auto settle = [&]() __attribute__((always_inline)) {
        while (ahead.b >= 0 && jb_after >= ahead.k1) {
            next_segment(ahead);
            jb_after = kBlock * wave;
        }
    };
    bool bad = false;
    if constexpr (RANGES) {
        settle();
        jseq = ahead.b;
        jb = jb_after;
        if (jseq >= 0) {
            ids[0] = read_ids(jseq, jb);
            const int L = ahead.L;
            jb_after += kStep;
            settle();
            if (ahead.b >= 0) ids_after = read_ids(ahead.b, jb_after);
            const Place a = place(L, jb, ids[0]);
            load(p.c.k, a, kr[0]);
            load(p.c.v, a, vr[0]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < D; i++) {
            const int key = key0 + kBlock * wave + i * kStep;
            if (key < seg.k1) {
                const Place a = place(seg.L, key, ids[i]);
                bad |= bad_page;
                load(p.c.k, a, kr[i]);
                load(p.c.v, a, vr[i]);
                ids[i] = read_ids(seg.b, key + D * kStep);
            }
        }
    }

    uint16_t * vw = reinterpret_cast<uint16_t *>(s_buf[wave]);
    const int v_rd = (4 * sgrp + (lane % 16) / 4) * VP + 4 * (lane % 4);
    auto wave_sync = [&]() {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    };

    for (;;) {
        const int L = max(seg.L, 0);
        int lim[QT];  // last key that the lane's row sees
#pragma unroll
        for (int t = 0; t < QT; t++)
            lim[t] = !row_ok(t) ? -1 : p.causal ? L - n_q + (rt * RT + 16 * t + srow) / G : L - 1;
        float m_run[QT], l_run[QT];  // of the lane's rows; l this lane's share
        float4_t o[QT][DT];          // O^T: lane holds O[16 t + srow][16 dt + 4 sgrp + v]
#pragma unroll
        for (int t = 0; t < QT; t++) {
            m_run[t] = kNegInf;
            l_run[t] = 0.f;
#pragma unroll
            for (int dt = 0; dt < DT; dt++) o[t][dt] = float4_t{0.f, 0.f, 0.f, 0.f};
        }
        bool q_raw = true;
        // one block of 32 keys from `key` on; next_k and next_v send for the keys and values that follow in its registers
        auto block = [&](const int key, u32x4 (&kr)[NL], u32x4 (&vr)[NL], auto && next_k, auto && next_v) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < NL; i++) *reinterpret_cast<u32x4 *>(vw + (KPL * i + vslot) * KPD + vcol) = kr[i];
            next_k();
            if (q_raw) {
                q_raw = false;
#pragma unroll
                for (int t = 0; t < QT; t++)
#pragma unroll
                    for (int ks = 0; ks < KS; ks++)
#pragma unroll
                        for (int e = 0; e < 4; e++) q[t][ks][e] = row_ok(t) ? (q[t][ks][e] & p.q_and) ^ p.q_xor : 0u;
            }
            wave_sync();
            // S^T = K Q^T, two tiles of 16 keys: lane holds keys 16 mt + 4 sgrp + v of its row
            const bool edge = key + kBlock > seg.k1 || (p.causal && key + kBlock > L - n_q + 1);
            float4_t sc[QT][2];
#pragma unroll
            for (int mt = 0; mt < 2; mt++) {
#pragma unroll
                for (int t = 0; t < QT; t++) sc[t][mt] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int ks = 0; ks < KS; ks++) {
                    const u32x4 k = *reinterpret_cast<const u32x4 *>(vw + (16 * mt + srow) * KPD + 32 * ks + 8 * sgrp);
#pragma unroll
                    for (int t = 0; t < QT; t++) sc[t][mt] = T::mfma16(k, q[t][ks], sc[t][mt]);
                }
            }
            u32x4 pb[QT];
#pragma unroll
            for (int t = 0; t < QT; t++) {
                float bmax = kNegInf;
#pragma unroll
                for (int mt = 0; mt < 2; mt++)
#pragma unroll
                    for (int v = 0; v < 4; v++) {
                        const int j = key + 16 * mt + 4 * sgrp + v;
                        sc[t][mt][v] = !edge || j <= lim[t] ? sc[t][mt][v] * p.scale_log2 : kNegInf;
                        bmax = fmaxf(bmax, sc[t][mt][v]);
                    }
                bmax = xor32_max(xor16_max(bmax));
                const float m_new = fmaxf(m_run[t], bmax);
                const bool none = m_new == kNegInf;  // no key yet: every exponent below is 2^-inf = 0
                const float m_use = none ? 0.f : m_new;
                const bool moved = m_new != m_run[t];
                const float corr = none ? 1.f : exp2_fast(m_run[t] - m_new);
                // P^T, rounded to T as the product takes both operands in one type; l sums the probabilities as they are, which
                // costs no unpacking (the outputs' error against 64 bits is 0.00173 in bf16, where 32-bit probabilities and the
                // output's rounding alone make 0.00165). Slot (sgrp, e) is key 16 (e / 4) + 4 sgrp + e % 4, the keys that the
                // transposing reads fetch.
                float bsum = 0.f;
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const float u = exp2_fast(sc[t][e / 4][e % 4] - m_use), w = exp2_fast(sc[t][e / 4][e % 4 + 1] - m_use);
                    bsum += u;
                    bsum += w;
                    pb[t][e / 2] = T::pack2(u, w);
                }
                l_run[t] = l_run[t] * corr + bsum;
                m_run[t] = m_new;
                if (__builtin_amdgcn_ballot_w64(moved)) {  // of some row
#pragma unroll
                    for (int dt = 0; dt < DT; dt++) o[t][dt] *= corr;
                }
            }
            wave_sync();  // the keys' reads are done
            if (edge) {
                // Values that some row must not see: behind the sequence's end they are zeros (the loads repeated the last
                // key); at keys that later rows see, an infinity or NaN (0 times it is NaN) is taken out of the product and
                // added to the rows that see it.
                bool odd = false;
#pragma unroll
                for (int i = 0; i < NL; i++) {
                    if (key + KPL * i + vslot >= L) vr[i] = u32x4{0u, 0u, 0u, 0u};
                    odd |= any_nonfinite<T>(vr[i]);
                }
                if (p.causal && n_q > 1 && __builtin_amdgcn_ballot_w64(odd)) {
#pragma unroll
                    for (int i = 0; i < NL; i++) *reinterpret_cast<u32x4 *>(vw + (KPL * i + vslot) * VP + vcol) = vr[i];
                    wave_sync();
#pragma unroll 1
                    for (int k = 0; k < kBlock; k++) {
#pragma unroll
                        for (int dt = 0; dt < DT; dt++) {
                            __builtin_amdgcn_sched_barrier(0);  // few masks at a time: this path must not cost the others registers
#pragma unroll
                            for (int v = 0; v < 4; v += 2) {
                                const uint32_t w = *reinterpret_cast<const uint32_t *>(vw + k * VP + 16 * dt + 4 * sgrp + v);
                                const float2 f = T::unpack2(w);
#pragma unroll
                                for (int t = 0; t < QT; t++) {
                                    if (key + k > lim[t]) continue;
                                    if ((w & T::kExp) == T::kExp) o[t][dt][v] += f.x;
                                    if (((w >> 16) & T::kExp) == T::kExp) o[t][dt][v + 1] += f.y;
                                }
                            }
                        }
                    }
                    wave_sync();
#pragma unroll
                    for (int i = 0; i < NL; i++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            uint32_t w = vr[i][e];
                            __builtin_amdgcn_sched_barrier(0);
                            if ((w & T::kExp) == T::kExp) w &= 0xffff0000u;
                            if (((w >> 16) & T::kExp) == T::kExp) w &= 0xffffu;
                            vr[i][e] = w;
                        }
                }
            }
#pragma unroll
            for (int i = 0; i < NL; i++) *reinterpret_cast<u32x4 *>(vw + (KPL * i + vslot) * VP + vcol) = vr[i];
            next_v();
            wave_sync();
            // O^T += V^T P^T
#pragma unroll
            for (int dt = 0; dt < DT; dt++) {
                const short4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) short4_t *)(vw + v_rd + 16 * dt));
                const short4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) short4_t *)(vw + v_rd + 16 * VP + 16 * dt));
                const u32x4 v = __builtin_bit_cast(u32x4, (short __attribute__((ext_vector_type(8)))){
                    lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
#pragma unroll
                for (int t = 0; t < QT; t++) o[t][dt] = T::mfma16(v, pb[t], o[t][dt]);
            }
            wave_sync();
        };
        if constexpr (RANGES) {
            while (jseq == seg.b) {
                // the next block: its keys into the registers that are free now, its values once this block's are in LDS; behind
                // it the page numbers of the one after, read ahead of its loads, so that a wait for them leaves those in flight
                Place a;
                const int key = jb;
                bad |= bad_page;
                jseq = ahead.b;
                jb = jb_after;
                const bool more = jseq >= 0;
                block(
                    key, kr[0], vr[0],
                    [&]() __attribute__((always_inline)) {
                        if (!more) return;
                        a = place(ahead.L, jb, ids_after);
                        jb_after += kStep;
                        settle();
                        if (ahead.b >= 0) ids_after = read_ids(ahead.b, jb_after);
                        __builtin_amdgcn_sched_barrier(0);
                        load(p.c.k, a, kr[0]);
                    },
                    [&]() __attribute__((always_inline)) {
                        if (more) load(p.c.v, a, vr[0]);
                    });
            }
        } else {
            for (int at = key0 + kBlock * wave; at < seg.k1; at += D * kStep) {
                static_for<0, D>([&](auto SC) __attribute__((always_inline)) {
                    constexpr int i = decltype(SC)::value;
                    const int key = at + i * kStep, next = key + D * kStep;
                    if (key >= seg.k1) return;
                    Place a;
                    block(
                        key, kr[i], vr[i],
                        [&]() __attribute__((always_inline)) {
                            if (next >= seg.k1) return;
                            a = place(seg.L, next, ids[i]);
                            bad |= bad_page;
                            ids[i] = read_ids(seg.b, next + D * kStep);
                            __builtin_amdgcn_sched_barrier(0);
                            load(p.c.k, a, kr[i]);
                        },
                        [&]() __attribute__((always_inline)) {
                            if (next < seg.k1) load(p.c.v, a, vr[i]);
                        });
                });
            }
        }
        const Seg done = seg;
        next_segment(seg);
        if (seg.b >= 0) load_q(seg.b);  // in flight over what follows

        // ---- join the waves; write the output, or publish this part ----
#pragma unroll
        for (int t = 0; t < QT; t++) {
            float l = xor32_add(xor16_add(l_run[t]));
            if (bad) l = __builtin_nanf("");
            if (sgrp == 0 && 16 * t + srow < RT) {
                s_m[wave][16 * t + srow] = m_run[t];  // -inf (weight 0) without a visible key
                s_l[wave][16 * t + srow] = l;
            }
            if (16 * t + srow < RT) {
#pragma unroll
                for (int dt = 0; dt < DT; dt++) *reinterpret_cast<float4_t *>(s_o(wave) + (16 * t + srow) * HD + 16 * dt + 4 * sgrp) = o[t][dt];
            }
        }
        lds_barrier();
        const int64_t row0 = (int64_t)done.b * n_q;  // the sequence's first query row
        const bool bad_len = done.L < 0;
        // an output quad: row i of the tile, dims d .. d + 4, weighted sum a over total tot at maximum M
        auto emit = [&](int i, int d, float4_t a, float M, float tot) __attribute__((always_inline)) {
            const int rr = rt * RT + i;
            if (rr >= p.rows) return;
            const int t = rr / G, h = g * G + rr % G;
            const bool empty = p.causal ? L - n_q + t < 0 : L == 0;  // no key: zeros (a length that is none: NaN)
            const float inv = 1.f / tot;
            float4_t w = empty ? float4_t{0.f, 0.f, 0.f, 0.f} : a * inv;
            if (bad_len) w = float4_t{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
            const int64_t at = (row0 + t) * p.out_stride + (int64_t)h * HD + d;
            if (p.out32) *reinterpret_cast<float4_t *>(static_cast<float *>(p.out) + at) = w;
            else *reinterpret_cast<u32x2 *>(static_cast<uint16_t *>(p.out) + at) = u32x2{T::pack2(w[0], w[1]), T::pack2(w[2], w[3])};
            if (d == 0 && p.lse) {
                const float v = empty ? kNegInf : (M + log2_fast(tot)) * kLn2;
                p.lse[(row0 + t) * p.n_head + h] = bad_len ? __builtin_nanf("") : v;
            }
        };
        // the parts of the sequence, and the slots of their partials (RANGES: two a range, for its first and its last segment)
        int ns, own, slot0, slot1, slot_step, counted;
        if constexpr (RANGES) {
            const int r0 = done.at / x.share, r1 = (done.at + quanta_of<kStep>(p, done.L) - 1) / x.share;
            ns = r1 - r0 + 1;
            own = r - r0;
            slot0 = 2 * r0 + (done.at > r0 * x.share ? 1 : 0);
            slot1 = 2 * r0 + 2;
            slot_step = 2;
            counted = r0;
        } else {
            ns = ch.n;
            own = ch.i;
            slot0 = ch.slot;
            slot1 = slot0 + 1;
            slot_step = 1;
            counted = ch.ordinal;
        }
        const int stride = (int)per_seq * SS;  // floats between slots
        float * part = p.part + tile * SS;
        const __amdgpu_buffer_rsrc_t rsrc = dev_rsrc(part);
        auto slot = [&](int k) { return (k == 0 ? slot0 : slot1 + (k - 1) * slot_step) * stride; };
        const int at_own = slot(own);
        for (int i = threadIdx.x; i < NQ; i += kThreads) {
            const int row = i / (HD / 4), d = 4 * (i % (HD / 4));
            if (rt * RT + row >= p.rows) continue;
            float mw[NW], M = kNegInf, tot = 0.f;
#pragma unroll
            for (int w = 0; w < NW; w++) mw[w] = s_m[w][row];
#pragma unroll
            for (int w = 0; w < NW; w++) M = fmaxf(M, mw[w]);
            const float Mu = M == kNegInf ? 0.f : M;
            float4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < NW; w++) {
                const float wt = exp2_fast(mw[w] - Mu);
                tot += s_l[w][row] * wt;
                acc += *reinterpret_cast<const float4_t *>(s_o(w) + row * HD + d) * wt;
            }
            if (ns == 1) {
                emit(row, d, acc, M, tot);
            } else {
                store16_dev(rsrc, 4 * (at_own + row * PR + d), acc);
                if (d == 0) publish2(part + at_own + row * PR + HD, M, tot);
            }
        }
        if (ns > 1) {
            // the partial is complete at device scope before it is counted in
            __builtin_amdgcn_s_waitcnt(0);
            __syncthreads();
            uint32_t * const counter = p.counters + (counted * per_seq + tile) * kCounterStride;
            if (threadIdx.x == 0)
                s_last = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)(ns - 1);
            __syncthreads();
            if (s_last) {
                __builtin_amdgcn_s_waitcnt(0);
                // ---- join the parts: weights 2^(m - M) of every (part, row), one lane per part, then the accumulator's quads, each
                // quad's parts striped over SF threads ----
                constexpr int SF = kThreads >= NQ ? kThreads / NQ : 1, CPT = NQ > kThreads ? NQ / kThreads : 1;
                // Parts of a quad in flight: as many as the registers hold (32 rows at head dim 128, 12 parts, 17.7 us with 8, 17.0
                // with 12). Past the last part the lanes load it again, or at head dim 64, whose launches have fewer parts, nothing
                // (7 parts 8.0 -> 7.55 us, but 32 parts at head dim 128 11.55 -> 11.75).
                constexpr int MC = CPT > 2 ? 4 : CPT == 2 ? 12 : 8;
                static_assert(kPagedMaxParts <= kWave, "one lane per part");
                static_assert((kPagedMaxParts * RT + 2 * RT) * 4 + (SF - 1) * NQ * 16 <= (int64_t)sizeof(s_buf), "merge scratch");
                float * s_w = reinterpret_cast<float *>(s_buf);                     // [part][row]
                float2 * s_row = reinterpret_cast<float2 *>(s_w + kPagedMaxParts * RT);  // (M, total)
                float4_t * s_acc = reinterpret_cast<float4_t *>(s_row + RT);        // [stripe - 1][quad]
                const int stripe = SF > 1 ? (int)threadIdx.x / NQ : 0;
                auto quad = [&](int c) { return SF > 1 ? (int)threadIdx.x % NQ : (int)threadIdx.x + c * kThreads; };
                // all rows' (m, l) of the wave and the first parts' quads are one round trip
                constexpr int WR = (RT + NW - 1) / NW;
                u32x2 ml[WR];
#pragma unroll
                for (int r = 0; r < WR; r++)
                    ml[r] = load8_dev(rsrc, 4 * (slot(min(lane, ns - 1)) + min(r * NW + wave, RT - 1) * PR + HD));
                u32x4 w[CPT][MC];
                auto fetch = [&](int s0) __attribute__((always_inline)) {
#pragma unroll
                    for (int c = 0; c < CPT; c++) {
                        const int i = quad(c), at = i / (HD / 4) * PR + 4 * (i % (HD / 4));
#pragma unroll
                        for (int e = 0; e < MC; e++) {
                            if (HD == 64 && s0 + SF * e >= ns) continue;
                            w[c][e] = load16_dev(rsrc, 4 * (at + slot(min(s0 + SF * e, ns - 1))));
                        }
                    }
                };
                fetch(stripe);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int r = 0; r < WR; r++) {
                    const int i = r * NW + wave;
                    if (i >= RT) break;
                    const float m = lane < ns ? __uint_as_float(ml[r][0]) : kNegInf;
                    const float M = row16_max(xor16_max(xor32_max(m)));
                    const float w = exp2_fast(m - (M == kNegInf ? 0.f : M));
                    const float tot = row16_sum(xor16_add(xor32_add(lane < ns ? __uint_as_float(ml[r][1]) * w : 0.f)));
                    if (lane < kPagedMaxParts) s_w[lane * RT + i] = w;
                    if (lane == 0) s_row[i] = make_float2(M, tot);
                }
                lds_barrier();  // the weights
                float4_t acc[CPT];
#pragma unroll
                for (int c = 0; c < CPT; c++) acc[c] = float4_t{0.f, 0.f, 0.f, 0.f};
                for (int s0 = stripe; s0 < ns; s0 += SF * MC) {
                    if (s0 != stripe) fetch(s0);
#pragma unroll
                    for (int c = 0; c < CPT; c++) {
                        const int i = quad(c) / (HD / 4);
#pragma unroll
                        for (int e = 0; e < MC; e++) {
                            const int k = s0 + SF * e;
                            if (k < ns) acc[c] += __builtin_bit_cast(float4_t, w[c][e]) * s_w[k * RT + i];
                        }
                    }
                }
                if constexpr (SF > 1) {
                    if (stripe > 0) s_acc[(stripe - 1) * NQ + quad(0)] = acc[0];
                    __syncthreads();
                    if (stripe == 0) {
#pragma unroll
                        for (int k = 1; k < SF; k++) acc[0] += s_acc[(k - 1) * NQ + quad(0)];
                    }
                }
                if (stripe == 0) {
#pragma unroll
                    for (int c = 0; c < CPT; c++) {
                        const int i = quad(c);
                        const float2 mt = s_row[i / (HD / 4)];
                        emit(i / (HD / 4), 4 * (i % (HD / 4)), acc[c], mt.x, mt.y);
                    }
                }
                if (threadIdx.x == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
        }
        if (seg.b < 0) break;
        bad = false;
        lds_barrier();  // the next segment's blocks go where the outputs were read from
    }
}

template <int HD, class T, int NW, bool RANGES>
void launch_rt(const PagedAttnParams & p, int rt, hipStream_t stream) {
    const int64_t groups = (int64_t)p.ranges * p.n_head_kv;
    const dim3 grid((uint32_t)(p.n_rowtiles == 1 ? groups : (groups + 7) / 8 * 8 * p.n_rowtiles)), block(NW * kWave);
    if (rt == 4) hipLaunchKernelGGL((paged_decode_kernel<HD, 4, T, NW, RANGES>), grid, block, 0, stream, p);
    else if (rt == 8) hipLaunchKernelGGL((paged_decode_kernel<HD, 8, T, NW, RANGES>), grid, block, 0, stream, p);
    else if (rt == 16) hipLaunchKernelGGL((paged_decode_kernel<HD, 16, T, NW, RANGES>), grid, block, 0, stream, p);
    else if constexpr (HD != 256) hipLaunchKernelGGL((paged_decode_kernel<HD, 32, T, NW, RANGES>), grid, block, 0, stream, p);
}

template <class T>
void launch_hd(const PagedAttnParams & p, int head_dim, int rt, int waves, hipStream_t stream) {
    if (head_dim == 256) {
        if (p.by_ranges) launch_rt<256, T, 4, true>(p, rt, stream);
        else launch_rt<256, T, 4, false>(p, rt, stream);
    } else if (head_dim == 64) {
        if (p.by_ranges) launch_rt<64, T, 4, true>(p, rt, stream);
        else if (waves == 8) launch_rt<64, T, 8, false>(p, rt, stream);
        else launch_rt<64, T, 4, false>(p, rt, stream);
    } else {
        if (p.by_ranges) launch_rt<128, T, 4, true>(p, rt, stream);
        else if (waves == 8) launch_rt<128, T, 8, false>(p, rt, stream);
        else launch_rt<128, T, 4, false>(p, rt, stream);
    }
}

}  // namespace

hipError_t launch_paged_decode(const PagedAttnParams & p, int head_dim, int dtype, int rt, int waves, hipStream_t stream) {
    if (dtype == 1) launch_hd<F16>(p, head_dim, rt, waves, stream);
    else launch_hd<BF16>(p, head_dim, rt, waves, stream);
    return hipGetLastError();
}

}  // namespace mx
