// Decode attention over a paged cache: a few new rows of each sequence, split over the sequences' lengths and joined.
//
// For row t of a sequence of L keys with n rows: s_j = scale q_t . k_j over keys j <= L - n + t (causal) or all L,
// out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m). Splits of the keys keep (m, l, acc) and are joined as
// M = max m, out = sum e^(m - M) acc / sum e^(m - M) l.
//
// What bounds it: each key and value is read once from HBM (the heads of a group and the sequence's rows share one pass), so
// long batches run at the memory's rate and short ones at the latency of a few dependent round trips.
//
//   * The lengths are in device memory, so that a captured launch replays while sequences grow: the grid is fixed by the host
//     and every workgroup works out its own part from the lengths. All waves read them (64 sequences a step) and agree on the
//     keys per split: the fewest with which the splits of all sequences fit the grid.
//   * A workgroup is one (sequence, kv head, split, tile of query rows). Each wave walks every NW-th block of 32 keys with the
//     next block in flight in registers; keys and values reach the operand layouts of v_mfma_f32_16x16x32 through LDS, values
//     through its transposing read, and the probabilities never leave registers.
//   * A page holds at least 16 keys, so the 16-key halves of a block each lie in one page: two page numbers per block, read one
//     block ahead of the keys they place.
//   * Splits publish their partials with device-scope stores and count themselves in; the last one of a tile joins them in
//     split order (the result does not depend on which was last) and resets the counter.
#include "mx_paged.hpp"

namespace mx {

namespace {

constexpr int kBlock = 32;      // keys a wave takes at a time
constexpr int kMaxSplits = 64;  // splits of a sequence at most (p.max_splits): one lane each in the merge

typedef short short4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ void publish2(float * p, float a, float b) {
    const uint64_t v = (uint64_t)__float_as_uint(a) | ((uint64_t)__float_as_uint(b) << 32);
    __hip_atomic_store(reinterpret_cast<uint64_t *>(p), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 collect2(const float * p) {
    const uint64_t v = __hip_atomic_load(reinterpret_cast<uint64_t *>(const_cast<float *>(p)), __ATOMIC_RELAXED,
                                         __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}

// What a workgroup takes, the same in all its waves.
struct Item {
    int32_t b;        // sequence, -1: nothing
    int32_t s, ns;    // split and splits of it
    int32_t len;      // its kv_len as it is
    int32_t chunk;    // keys per split
    int32_t ordinal;  // split sequences before it
    int32_t slot;     // splits of those
};

// The `j`-th (sequence, split) pair of the launch, for splits in multiples of Q keys.
template <int Q>
__device__ __forceinline__ Item find_item(const PagedAttnParams & p, int j, int lane) {
    const int n_seq = p.c.n_seq;
    const int len0 = p.c.kv_len[min(lane, n_seq - 1)];
    auto len_of = [&](int base) { return base == 0 ? len0 : p.c.kv_len[min(base + lane, n_seq - 1)]; };
    auto quanta = [&](int base, int len) {
        return base + lane < n_seq && length_ok(p.c, len) ? (len + Q - 1) / Q : 0;
    };
    float sum = 0.f;  // of quanta: only the plan depends on it
    int most = 0;
    for (int base = 0; base < n_seq; base += kWave) {
        const int n = quanta(base, len_of(base));
        sum += (float)n;
        most = max(most, n);
    }
    sum = wave_sum(sum);
    most = max(1, wave_imax(most));
    auto splits = [&](int base, int len, int c) {  // an empty sequence is one split: its rows are written too
        return base + lane < n_seq ? max(1, (quanta(base, len) + c - 1) / c) : 0;
    };
    auto count = [&](int c) {
        int r = 0;
        for (int base = 0; base < n_seq; base += kWave) r += splits(base, len_of(base), c);
        return wave_isum(r);
    };
    // the shortest splits that the grid has room for: between an equal share of the work and one that surely fits
    const int extra = p.budget - n_seq;
    int c = max((most + p.max_splits - 1) / p.max_splits, (int)fminf(ceilf(sum / (float)p.budget), (float)most));
    if (n_seq == 1) {
        c = max(c, (most + p.budget - 1) / p.budget);
    } else if (count(c) > p.budget) {
        int lo = c, hi = most;  // count(lo) is too many; whole sequences are n_seq
        if (extra > 0) hi = max(lo + 1, min(most, (int)fminf(sum / (float)extra, (float)most) + 1));
        if (hi < most && count(hi) > p.budget) hi = most;  // the float sum was rounded down
        for (int i = 0; i < 4 && hi - lo > 1 && (hi - lo) * 16 > lo; i++) {
            const int mid = (lo + hi) / 2;
            if (count(mid) > p.budget) lo = mid;
            else hi = mid;
        }
        c = hi;
    }
    Item it{-1, 0, 1, 0, c * Q, 0, 0};
    int before = 0, ordinal = 0;
    for (int base = 0; base < n_seq; base += kWave) {
        const int len = len_of(base), ns = splits(base, len, c);
        const int upto = before + wave_iscan(ns);
        const uint64_t many = __builtin_amdgcn_ballot_w64(ns > 1);
        const uint64_t past = __builtin_amdgcn_ballot_w64(upto > j);
        if (past) {
            const int l = __builtin_ctzll(past);
            it.b = base + l;
            it.ns = __builtin_amdgcn_readlane(ns, l);
            it.len = __builtin_amdgcn_readlane(len, l);
            const int first = __builtin_amdgcn_readlane(upto, l) - it.ns;
            it.s = j - first;
            it.ordinal = ordinal + __builtin_popcountll(many & ((1ull << l) - 1));
            it.slot = first - (it.b - it.ordinal);  // the sequences before it that are not split have one each
            return it;
        }
        before = __builtin_amdgcn_readlane(upto, 63);
        ordinal += __builtin_popcountll(many);
    }
    return it;
}

// HD: head_dim. RT: query rows per tile (4, 8 or 16; the matrix products always have 16, the others are zero). T: type of
// pages and query rows. NW: waves.
template <int HD, int RT, class T, int NW>
__global__ __launch_bounds__(NW * kWave) __attribute__((amdgpu_waves_per_eu(HD == 128 || NW == 8 ? 2 : 1)))
void paged_decode_kernel(PagedAttnParams p) {
    constexpr int KS = HD / 32;          // product steps along head_dim
    constexpr int LPR = HD / 8;          // lanes per key row
    constexpr int KPL = kWave / LPR;     // key rows per load
    constexpr int NL = kBlock / KPL;     // loads per lane per block, for each of keys and values
    constexpr int VP = HD + 16;          // LDS row pitch of a block's values (conflict-free transposing reads) ...
    constexpr int KPD = HD + 8;          // ... and keys, which pass through the same LDS first
    constexpr int DT = HD / 16;
    constexpr int kThreads = NW * kWave;
    constexpr int PR = HD + 4;           // floats of a partial's row: acc, m, l
    static_assert(16 % KPL == 0, "a load's rows lie in one page");
    static_assert(RT * HD * 4 <= kBlock * VP * 2, "a wave's outputs reuse its values' LDS");
    __shared__ uint16_t s_v[NW][kBlock * VP];
    __shared__ float s_m[NW][RT], s_l[NW][RT];
    __shared__ int s_last;
    auto s_o = [&](int w) { return reinterpret_cast<float *>(s_v[w]); };

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
    // kv heads fastest (workgroups are dealt to the 8 XCDs round-robin), the row tiles of one split on one XCD, 8 ids apart:
    // all but the first find its keys in that XCD's L2
    const uint32_t id = blockIdx.x, tiles = p.n_rowtiles;
    const uint32_t grp = id / (8 * tiles) * 8 + id % 8;
    const int rt = id / 8 % tiles, g = grp % p.n_head_kv, j = grp / p.n_head_kv;
    const Item it = find_item<NW * kBlock>(p, j, lane);
    if (it.b < 0) return;  // uniform over the workgroup
    const int G = p.group, n_q = p.n_q;
    const int64_t row0 = (int64_t)it.b * n_q;  // the sequence's first query row
    const bool bad_len = !length_ok(p.c, it.len);
    const int L = bad_len ? 0 : it.len;

    // an output quad: row r of the tile, dims d .. d + 4, weighted sum a over total tot at maximum M
    auto emit = [&](int r, int d, float4_t a, float M, float tot) __attribute__((always_inline)) {
        const int rr = rt * RT + r;
        if (rr >= p.rows) return;
        const int t = rr / G, h = g * G + rr % G;
        const bool empty = p.causal ? L - n_q + t < 0 : L == 0;  // no key: zeros (a length that is none: NaN)
        const float inv = 1.f / tot;
        float4_t o = empty ? float4_t{0.f, 0.f, 0.f, 0.f} : a * inv;
        if (bad_len) o = float4_t{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
        const int64_t off = (row0 + t) * p.out_stride + (int64_t)h * HD + d;
        if (p.out32) *reinterpret_cast<float4_t *>(static_cast<float *>(p.out) + off) = o;
        else *reinterpret_cast<u32x2 *>(static_cast<uint16_t *>(p.out) + off) = u32x2{T::pack2(o[0], o[1]), T::pack2(o[2], o[3])};
        if (d == 0 && p.lse) {
            const float v = empty ? kNegInf : (M + log2_fast(tot)) * kLn2;
            p.lse[(row0 + t) * p.n_head + h] = bad_len ? __builtin_nanf("") : v;
        }
    };
    if (L == 0) {
        for (int i = threadIdx.x; i < RT * HD / 4; i += kThreads)
            emit(i / (HD / 4), 4 * (i % (HD / 4)), float4_t{0.f, 0.f, 0.f, 0.f}, 0.f, 1.f);
        return;
    }
    const int j0 = it.s * it.chunk, j1 = min(j0 + it.chunk, L);
    const int srow = lane % 16, sgrp = lane / 16;           // score lanes: query row, keys 4 sgrp .. + 4 of a 16-key tile
    const int vslot = lane / LPR, vcol = 8 * (lane % LPR);  // load lanes: key row, first dim
    const int32_t * table = p.c.table + it.b * p.c.table_stride;
    const uint16_t * kg = p.c.k + (int64_t)g * p.c.head_stride + vcol;
    const uint16_t * vg = p.c.v + (int64_t)g * p.c.head_stride + vcol;
    const int page_mask = (1 << p.c.page_shift) - 1;
    const uint32_t kv_stride = (uint32_t)p.c.kv_stride;

    // page numbers of a block's two halves, in lanes 0 and 1 (halves behind the last key: the last key's page)
    auto read_ids = [&](int jb) { return table[min(jb + 16 * (lane & 1), L - 1) >> p.c.page_shift]; };
    bool bad = false;
    struct Block {
        u32x4 k[NL], v[NL];
    };
    auto load_block = [&](int jb, int ids, Block & blk) __attribute__((always_inline)) {
        int64_t base[2];
        int last[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            int id = __builtin_amdgcn_readlane(ids, h);
            const bool ok = page_ok(p.c, id);
            bad |= !ok;
            id = ok ? id : 0;
            const int k16 = min(jb + 16 * h, (L - 1) & ~15);
            base[h] = (int64_t)id * p.c.page_stride + (int64_t)(k16 & page_mask) * p.c.kv_stride;
            last[h] = L - 1 - k16;
        }
#pragma unroll
        for (int i = 0; i < NL; i++) {
            const int h = KPL * i / 16, r = min(KPL * i % 16 + vslot, last[h]);
            blk.k[i] = load16(kg + base[h] + (uint32_t)r * kv_stride);
        }
#pragma unroll
        for (int i = 0; i < NL; i++) {
            const int h = KPL * i / 16, r = min(KPL * i % 16 + vslot, last[h]);
            blk.v[i] = load16(vg + base[h] + (uint32_t)r * kv_stride);
        }
    };

    int jb = j0 + kBlock * wave;
    const int ids0 = read_ids(jb);
    int ids = read_ids(jb + kBlock * NW);
    Block cur, nxt;
    load_block(jb, ids0, cur);
    // this lane's query operand (a row past the tile: the problem's first row, zeroed)
    const int rr = rt * RT + srow;
    const bool row_ok = srow < RT && rr < p.rows;
    const int st = row_ok ? rr / G : 0, sh = g * G + (row_ok ? rr % G : 0);
    const int lim = !row_ok ? -1 : p.causal ? L - n_q + st : L - 1;  // last key that the row sees
    u32x4 q[KS];
    {
        const uint16_t * qr = p.q + (row0 + st) * p.q_stride + (int64_t)sh * HD + 8 * sgrp;
#pragma unroll
        for (int ks = 0; ks < KS; ks++) q[ks] = load16(qr + 32 * ks);
    }
    const uint32_t q_and = row_ok ? p.q_and : 0u, q_xor = row_ok ? p.q_xor : 0u;
    bool q_raw = true;

    float m_run = kNegInf, l_run = 0.f;  // of row srow; l this lane's share
    float4_t o[DT];                      // O^T: lane holds O[srow][16 dt + 4 sgrp + v]
#pragma unroll
    for (int dt = 0; dt < DT; dt++) o[dt] = float4_t{0.f, 0.f, 0.f, 0.f};
    uint16_t * vw = s_v[wave];
    const int v_rd = (4 * sgrp + (lane % 16) / 4) * VP + 4 * (lane % 4);
    auto wave_sync = [&]() {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    };

    for (; jb < j1; jb += kBlock * NW) {
        const int jn = jb + kBlock * NW;
        if (jn < j1) {
            const int now = ids;
            ids = read_ids(jn + kBlock * NW);  // ahead of the block's loads: a wait for it leaves those in flight
            __builtin_amdgcn_sched_barrier(0);
            load_block(jn, now, nxt);
        }
        if (q_raw) {
            q_raw = false;
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int e = 0; e < 4; e++) q[ks][e] = (q[ks][e] & q_and) ^ q_xor;
        }
#pragma unroll
        for (int i = 0; i < NL; i++) *reinterpret_cast<u32x4 *>(vw + (KPL * i + vslot) * KPD + vcol) = cur.k[i];
        wave_sync();
        // S^T = K Q^T, two tiles of 16 keys: lane holds keys 16 mt + 4 sgrp + v of row srow
        float sc[2][4];
        const bool edge = jb + kBlock > j1 || (p.causal && jb + kBlock > L - n_q + 1);
#pragma unroll
        for (int mt = 0; mt < 2; mt++) {
            float4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
                acc = T::mfma16(*reinterpret_cast<const u32x4 *>(vw + (16 * mt + srow) * KPD + 32 * ks + 8 * sgrp), q[ks], acc);
#pragma unroll
            for (int v = 0; v < 4; v++) {
                const int key = jb + 16 * mt + 4 * sgrp + v;
                sc[mt][v] = !edge || key <= lim ? acc[v] * p.scale_log2 : kNegInf;
            }
        }
        float bmax = kNegInf;
#pragma unroll
        for (int mt = 0; mt < 2; mt++)
#pragma unroll
            for (int v = 0; v < 4; v++) bmax = fmaxf(bmax, sc[mt][v]);
        bmax = xor32_max(xor16_max(bmax));
        const float m_new = fmaxf(m_run, bmax);
        const bool none = m_new == kNegInf;      // no key yet: every exponent below is 2^-inf = 0
        const float m_use = none ? 0.f : m_new;
        const float corr = none ? 1.f : exp2_fast(m_run - m_new);
        // P^T, rounded to T for the product; l sums the probabilities as they are. Slot (sgrp, e) is key
        // 16 (e / 4) + 4 sgrp + e % 4, the keys that the transposing reads fetch.
        u32x4 pb;
        float bsum = 0.f;
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const float a = exp2_fast(sc[e / 4][e % 4] - m_use), b = exp2_fast(sc[e / 4][e % 4 + 1] - m_use);
            bsum += a;
            bsum += b;
            pb[e / 2] = T::pack2(a, b);
        }
        l_run = l_run * corr + bsum;
        m_run = m_new;
#pragma unroll
        for (int dt = 0; dt < DT; dt++) o[dt] *= corr;
        wave_sync();  // the keys' reads are done
        if (edge) {
            // Values that some row must not see: behind the sequence's end they are zeros (the loads repeated the last
            // key); at keys that later rows see, an infinity or NaN (0 times it is NaN) is taken out of the product and added
            // to the rows that see it.
            bool odd = false;
#pragma unroll
            for (int i = 0; i < NL; i++) {
                if (jb + KPL * i + vslot >= L) cur.v[i] = u32x4{0u, 0u, 0u, 0u};
                odd |= any_nonfinite<T>(cur.v[i]);
            }
            if (p.causal && n_q > 1 && __builtin_amdgcn_ballot_w64(odd)) {
#pragma unroll
                for (int i = 0; i < NL; i++) *reinterpret_cast<u32x4 *>(vw + (KPL * i + vslot) * VP + vcol) = cur.v[i];
                wave_sync();
                for (int k = 0; k < kBlock; k++) {
                    if (jb + k > lim) continue;
#pragma unroll
                    for (int dt = 0; dt < DT; dt++)
#pragma unroll
                        for (int v = 0; v < 4; v += 2) {
                            const uint32_t w = *reinterpret_cast<const uint32_t *>(vw + k * VP + 16 * dt + 4 * sgrp + v);
                            const float2 x = T::unpack2(w);
                            if ((w & T::kExp) == T::kExp) o[dt][v] += x.x;
                            if (((w >> 16) & T::kExp) == T::kExp) o[dt][v + 1] += x.y;
                        }
                }
                wave_sync();
#pragma unroll
                for (int i = 0; i < NL; i++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        uint32_t w = cur.v[i][e];
                        if ((w & T::kExp) == T::kExp) w &= 0xffff0000u;
                        if (((w >> 16) & T::kExp) == T::kExp) w &= 0xffffu;
                        cur.v[i][e] = w;
                    }
            }
        }
#pragma unroll
        for (int i = 0; i < NL; i++) *reinterpret_cast<u32x4 *>(vw + (KPL * i + vslot) * VP + vcol) = cur.v[i];
        wave_sync();
        // O^T += V^T P^T
#pragma unroll
        for (int dt = 0; dt < DT; dt++) {
            const short4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) short4_t *)(vw + v_rd + 16 * dt));
            const short4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) short4_t *)(vw + v_rd + 16 * VP + 16 * dt));
            const u32x4 a = __builtin_bit_cast(u32x4, (short __attribute__((ext_vector_type(8)))){
                lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
            o[dt] = T::mfma16(a, pb, o[dt]);
        }
        wave_sync();
        cur = nxt;
    }

    l_run = xor32_add(xor16_add(l_run));
    if (bad) l_run = __builtin_nanf("");
    if (lane < RT) {
        s_m[wave][lane] = m_run;  // -inf (weight 0) without a visible key
        s_l[wave][lane] = l_run;
    }
    if (srow < RT) {
#pragma unroll
        for (int dt = 0; dt < DT; dt++) *reinterpret_cast<float4_t *>(s_o(wave) + srow * HD + 16 * dt + 4 * sgrp) = o[dt];
    }
    __syncthreads();

    // ---- join the waves; write the output, or publish this split's partial ----
    constexpr int NQ = RT * HD / 4;  // output quads of the tile
    constexpr int64_t SS = (int64_t)RT * PR;
    const int64_t tile = (int64_t)rt * p.n_head_kv + g, per_seq = (int64_t)p.n_head_kv * p.n_rowtiles;
    float * part = p.part + ((int64_t)it.slot * per_seq + tile * it.ns) * SS;  // the tile's first split
    const __amdgpu_buffer_rsrc_t rsrc = dev_rsrc(part);
    const bool single = it.ns == 1;
    for (int i = threadIdx.x; i < NQ; i += kThreads) {
        const int r = i / (HD / 4), d = 4 * (i % (HD / 4));
        if (rt * RT + r >= p.rows) continue;
        float mw[NW], M = kNegInf, tot = 0.f;
#pragma unroll
        for (int w = 0; w < NW; w++) mw[w] = s_m[w][r];
#pragma unroll
        for (int w = 0; w < NW; w++) M = fmaxf(M, mw[w]);
        const float Mu = M == kNegInf ? 0.f : M;
        float4_t a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const float wt = exp2_fast(mw[w] - Mu);
            tot += s_l[w][r] * wt;
            a += *reinterpret_cast<const float4_t *>(s_o(w) + r * HD + d) * wt;
        }
        if (single) {
            emit(r, d, a, M, tot);
        } else {
            store16_dev(rsrc, (int)(4 * (it.s * SS + r * PR + d)), a);
            if (d == 0) publish2(part + it.s * SS + r * PR + HD, M, tot);
        }
    }
    if (single) return;
    // the partial is complete at device scope before it is counted in
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    uint32_t * const counter = p.counters + ((int64_t)it.ordinal * per_seq + tile) * kCounterStride;
    if (threadIdx.x == 0)
        s_last = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)(it.ns - 1);
    __syncthreads();
    if (!s_last) return;
    __builtin_amdgcn_s_waitcnt(0);

    // ---- join the splits: weights 2^(m - M) of every (split, row), one lane per split, then the accumulator's quads, each
    // quad's splits striped over SF threads ----
    constexpr int SF = kThreads >= NQ ? kThreads / NQ : 1, CPT = NQ > kThreads ? NQ / kThreads : 1;
    constexpr int MC = CPT > 1 ? 4 : 8;  // splits of a quad in flight
    static_assert(kMaxSplits <= kWave, "one lane per split");
    static_assert((kMaxSplits * RT + 2 * RT) * 4 + (SF - 1) * NQ * 16 <= (int64_t)sizeof(s_v), "merge scratch");
    float * s_w = reinterpret_cast<float *>(s_v);                        // [split][row]
    float2 * s_row = reinterpret_cast<float2 *>(s_w + kMaxSplits * RT);  // (M, total)
    float4_t * s_acc = reinterpret_cast<float4_t *>(s_row + RT);         // [stripe - 1][quad]
    const int ns = it.ns, stripe = SF > 1 ? (int)threadIdx.x / NQ : 0;
    auto quad = [&](int c) { return SF > 1 ? (int)threadIdx.x % NQ : (int)threadIdx.x + c * kThreads; };
#pragma unroll
    for (int r0 = 0; r0 < RT; r0 += NW) {
        const int r = r0 + wave;
        if (r >= RT) break;
        const float2 ml = collect2(part + min(lane, ns - 1) * SS + r * PR + HD);
        const float m = lane < ns ? ml.x : kNegInf;
        const float M = row16_max(xor16_max(xor32_max(m)));
        const float w = exp2_fast(m - (M == kNegInf ? 0.f : M));
        const float tot = row16_sum(xor16_add(xor32_add(lane < ns ? ml.y * w : 0.f)));
        if (lane < kMaxSplits) s_w[lane * RT + r] = w;
        if (lane == 0) s_row[r] = make_float2(M, tot);
    }
    float4_t acc[CPT];
#pragma unroll
    for (int c = 0; c < CPT; c++) acc[c] = float4_t{0.f, 0.f, 0.f, 0.f};
    bool first = true;
    for (int s0 = stripe; s0 < ns || first; s0 += SF * MC) {
        u32x4 x[CPT][MC];
#pragma unroll
        for (int c = 0; c < CPT; c++) {
            const int i = quad(c), at = i / (HD / 4) * PR + 4 * (i % (HD / 4));
#pragma unroll
            for (int e = 0; e < MC; e++) x[c][e] = load16_dev(rsrc, 4 * (int)(at + min(s0 + SF * e, ns - 1) * SS));
        }
        if (first) __syncthreads();  // the weights
        first = false;
#pragma unroll
        for (int c = 0; c < CPT; c++) {
            const int r = quad(c) / (HD / 4);
#pragma unroll
            for (int e = 0; e < MC; e++) {
                const int k = s0 + SF * e;
                if (k < ns) acc[c] += __builtin_bit_cast(float4_t, x[c][e]) * s_w[k * RT + r];
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

template <int HD, class T, int NW>
void launch_rt(const PagedAttnParams & p, int rt, hipStream_t stream) {
    const int64_t groups = (int64_t)p.budget * p.n_head_kv;
    const dim3 grid((uint32_t)(p.n_rowtiles == 1 ? groups : (groups + 7) / 8 * 8 * p.n_rowtiles)), block(NW * kWave);
    if (rt == 4) hipLaunchKernelGGL((paged_decode_kernel<HD, 4, T, NW>), grid, block, 0, stream, p);
    else if (rt == 8) hipLaunchKernelGGL((paged_decode_kernel<HD, 8, T, NW>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((paged_decode_kernel<HD, 16, T, NW>), grid, block, 0, stream, p);
}

template <class T>
void launch_hd(const PagedAttnParams & p, int head_dim, int rt, int waves, hipStream_t stream) {
    if (head_dim == 256) launch_rt<256, T, 4>(p, rt, stream);
    else if (head_dim == 64 && waves == 8) launch_rt<64, T, 8>(p, rt, stream);
    else if (head_dim == 64) launch_rt<64, T, 4>(p, rt, stream);
    else if (waves == 8) launch_rt<128, T, 8>(p, rt, stream);
    else launch_rt<128, T, 4>(p, rt, stream);
}

}  // namespace

hipError_t launch_paged_decode(const PagedAttnParams & p, int head_dim, int dtype, int rt, int waves, hipStream_t stream) {
    if (dtype == 1) launch_hd<F16>(p, head_dim, rt, waves, stream);
    else launch_hd<BF16>(p, head_dim, rt, waves, stream);
    return hipGetLastError();
}

}  // namespace mx
