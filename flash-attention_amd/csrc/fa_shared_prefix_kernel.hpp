// Attention of a batch whose requests share a long prefix, over a paged K/V cache.  Row (t, h), token t of request b and
// query head h of K/V head h / g:
//     O = sum_j p_j V_j / sum_j p_j,   p_j = exp(scale Q.K_j),   j over the Lp keys of the prefix and over the request's
//     own keys j <= k_len[b] - n[b] + (t - q_start[b])  (causal; all k_len[b] of them otherwise).
// The sum over j falls into parts that are computed apart and joined by their maxima (log-sum-exp): the prefix part is one
// matrix product for the whole batch, its rows being the g heads of ALL tokens stacked up against each K/V head, so the
// prefix is read from memory once per 128 stacked rows instead of once per request; the own part has the rows of one
// request.  Both parts are divided over ranges of keys until the chip is full.
// Both products are transposed (S^T = K.Q^T; the score registers, rounded to the cache's type, are the B operand of
// O^T += V^T.P^T), scores, maxima, sums and O are 32-bit.  P is rounded once, as every matrix product's operand must be; its
// sum l is taken before that.  A workgroup has one of two forms: shared_few_rows (bound by reading K and V) and
// shared_many_rows (matrix products; what bounds it stands there), chosen by the number of rows.
// fa_shared_prefix_merge_kernel joins the parts.
//
// Measured (one MI355X, kernels alone under the profiler, profiles/paged_forms.txt; 8 K/V heads of 4; a large copy moves 4.9 TB/s, a
// large matrix product runs at 1.3 PFLOP/s), D = 64 / 128 / 256:
//   one token of each of 128 requests, up to 1 024 own keys: 3.3 / 4.4 / 4.4 TB/s; up to 2 048: 4.2 / 4.8 / 5.1;
//   8 prompts of up to 2 048 tokens behind 8 192 keys: 692 / 912 / 921 TFLOP/s; one of 4 096 against itself: 515 / 724 / 724;
//   256 stacked tokens behind 16 384 keys: 364 / 564 / 552 TFLOP/s.
//
// Masks.  A tile that holds a masked place for some row of the wave (the end of the range, the causal diagonal, a page that
// is none) takes the masked form of the step: scores of masked places become -inf whatever K holds there, and V is
// multiplied with its infinities and NaN taken out (0 x NaN is NaN), which are then added to the rows that do see them.
// Rows that see no key give 0.
#pragma once
#include "fa_fwd_general_kernel.hpp"
#include "fa_fwd_ring_kernel.hpp"  // wait_all_vmem
#include "fa_cache_kernels.hpp"  // wave_sum_up
#include "fa_owned_acc.hpp"
#include "fa_paged_index.hpp"

namespace fa {

struct SharedPrefixParams {
    const uint16_t* q;
    uint16_t* o;
    const uint16_t* kc;
    const uint16_t* vc;
    int64_t q_tok, q_head, o_tok, o_head;
    CacheStrides ks, vs;
    const int* prefix_table;
    const int* block_table;
    int64_t table_stride;
    const int* q_start;
    const int* k_len;
    float* part_o;    // [parts][T * Hq][D], un-normalised
    float* part_ml;   // [parts][T * Hq][2]: largest score (log2 units) and sum of exp2(score - largest)
    int* row_parts;   // [T * Hq]: parts of the row's sum; 0: its output is written already
    int T, B, Hkv, g, log2_page, n_pages, prefix_len, table_width, causal;
    float scale_log2e;
    DivisionRule rule;
    unsigned g_reciprocal;  // 2^32 / g, rounded up
};

template <typename E>
struct Elem;
template <>
struct Elem<_Float16> {
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    typedef _Float16 v4 __attribute__((ext_vector_type(4)));
    static constexpr unsigned kExpMask = 0x7c00;
    static __device__ __forceinline__ f32x16 mfma(v8 a, v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ f32x4 mfma16(v8 a, v8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ f32x4 mfma16(v4 a, v4 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x16f16(a, b, c, 0, 0, 0); }
    template <int LO>  // a[LO : LO + 15] += a.b
    static __device__ __forceinline__ void mfma_owned(v8 a, v8 b) {
        asm volatile("v_mfma_f32_32x32x16_f16 a[%2:%3], %0, %1, a[%2:%3]" : : "v"(a), "v"(b), "n"(LO), "n"(LO + 15));
    }
};
template <>
struct Elem<__bf16> {
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    typedef __bf16 v4 __attribute__((ext_vector_type(4)));
    static constexpr unsigned kExpMask = 0x7f80;
    static __device__ __forceinline__ f32x16 mfma(v8 a, v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ f32x4 mfma16(v8 a, v8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ f32x4 mfma16(v4 a, v4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(short4_t, a), __builtin_bit_cast(short4_t, b), c, 0, 0, 0);
    }
    template <int LO>
    static __device__ __forceinline__ void mfma_owned(v8 a, v8 b) {
        asm volatile("v_mfma_f32_32x32x16_bf16 a[%2:%3], %0, %1, a[%2:%3]" : : "v"(a), "v"(b), "n"(LO), "n"(LO + 15));
    }
};

// max that keeps NaN (v_maximum3_f32): a row that sees a NaN score is NaN, and no operand is canonicalised first.
__device__ __forceinline__ float max_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// Infinities and NaN of a V fragment (4 or 8 elements): taken out (returned fragment), and their places (kind 1 NaN, 2 +inf,
// 3 -inf) as ones.
template <typename E, typename V>
__device__ __forceinline__ V finite_part(V x, bool& special) {
    constexpr int W = sizeof(V) / 4;
    typedef unsigned words __attribute__((ext_vector_type(W)));
    words u = __builtin_bit_cast(words, x);
    constexpr unsigned m = Elem<E>::kExpMask;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        if ((u[i] & m) == m) u[i] &= 0xffff0000u, special = true;
        if ((u[i] & (m << 16)) == m << 16) u[i] &= 0x0000ffffu, special = true;
    }
    return __builtin_bit_cast(V, u);
}
template <typename E, typename V>
__device__ __forceinline__ V special_part(V x, int kind) {
    constexpr int W = sizeof(V) / 4;
    typedef unsigned words __attribute__((ext_vector_type(W)));
    const words u = __builtin_bit_cast(words, x);
    constexpr unsigned m = Elem<E>::kExpMask;
    V r;
#pragma unroll
    for (int i = 0; i < 2 * W; ++i) {
        const unsigned h = (u[i / 2] >> (16 * (i & 1))) & 0xffffu, a = h & 0x7fffu;
        const int k = a > m ? 1 : a < m ? 0 : h == a ? 2 : 3;
        r[i] = (E)(k == kind ? 1.0f : 0.0f);
    }
    return r;
}
__device__ __forceinline__ float special_value(int kind) {
    return __builtin_bit_cast(float, kind == 1 ? 0x7fc00000u : kind == 2 ? 0x7f800000u : 0xff800000u);
}

template <int D>
struct SharedCfg;
template <>
struct SharedCfg<64> {
    static constexpr int kTk = key_tile(64), kStages = 4, kFewBlocks = 2;  // 16 KiB a stage
};
template <>
struct SharedCfg<128> {
    static constexpr int kTk = key_tile(128), kStages = 4, kFewBlocks = 1;  // 16 KiB
};
template <>
struct SharedCfg<256> {
    static constexpr int kTk = key_tile(256), kStages = 4, kFewBlocks = 1;  // 32 KiB
};

// The division of a launch into workgroups (SharedPlan), from the requests' lengths; every wave computes it for itself (no
// barrier: all write the same numbers to LDS, each reads what it has written).  That is one round of loads for every 128 requests
// and two of lane sums for every 64, in each of about B x Hkv workgroups: nothing beside 128 requests' keys (one token each, up to 128
// own keys, 32 heads on 8: 26 us), more than the keys from some 500 on (512: 155 us, 1 000: 444, 2 000: 1 484, 4 000: 5 459).

// LDS, until the first transfer: per request its first token, its own keys, the stacked tokens and the items before it.
struct SharedTables {
    int *tok0, *keys, *stacked, *items;
    __device__ __forceinline__ SharedTables(char* lds, int B) {
        tok0 = reinterpret_cast<int*>(lds);
        keys = tok0 + B + 1;
        stacked = keys + B;
        items = stacked + B;
    }
};

// From here on a lane reads what other lanes of its wave wrote to LDS before.  A wave's LDS operations complete in order; this holds
// the compiler to the order written.
__device__ __forceinline__ void wave_exchange() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_float(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, true));
}
__device__ __forceinline__ float wave_total(float v) {
    v += dpp_float<0x111, 0xf>(v);
    v += dpp_float<0x112, 0xf>(v);
    v += dpp_float<0x114, 0xf>(v);
    v += dpp_float<0x118, 0xf>(v);
    v += dpp_float<0x142, 0xa>(v);
    v += dpp_float<0x143, 0xc>(v);
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}
struct HardwareRcp {
    __device__ __forceinline__ float operator()(int b) const { return __builtin_amdgcn_rcpf((float)b); }
};
// R / g for the rows of a launch (R g < 2^32: the launcher's check), by the reciprocal 2^32 / g rounded up.
__device__ __forceinline__ int div_group(const SharedPrefixParams& p, int R) { return p.g == 1 ? R : (int)__umulhi((unsigned)R, p.g_reciprocal); }

// Returns the number of items.
template <int TK>
__device__ __forceinline__ int shared_plan(const SharedPrefixParams& p, SharedPlan& s, const SharedTables& tab) {
    const int lane = threadIdx.x & 63;
    const int prefix_tiles = (p.prefix_len + TK - 1) / TK;
    int tokens = 0;
    LaunchWork work;
    for (int b0 = 0; b0 < p.B; b0 += 128) {
        int q0[2], q1[2], k[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int b = min(b0 + 64 * i + lane, p.B - 1);
            q0[i] = p.q_start[b], q1[i] = p.q_start[b + 1], k[i] = p.k_len[b];
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (b0 + 64 * i >= p.B) break;
            const int b = b0 + 64 * i + lane;
            const int tok0 = clamp_int(q0[i], 0, p.T), keys = clamp_int(k[i], 0, p.table_width << p.log2_page);
            const int n = b < p.B ? clamp_int(q1[i], tok0, p.T) - tok0 : 0, rows = n * p.g, own = (keys + TK - 1) / TK;
            const int stacked = rows < kRowTile ? n : 0, sum = wave_sum_up(stacked);
            if (b < p.B) {
                tab.tok0[b] = tok0;
                tab.keys[b] = keys;
                tab.stacked[b] = tokens + sum - stacked;
                if (b == p.B - 1) tab.tok0[p.B] = tok0 + n;
                work.add_request(p.rule, rows, own, prefix_tiles);
            }
            tokens += __builtin_amdgcn_readlane(sum, 63);
        }
    }
    wave_exchange();
    work.few = wave_total(work.few), work.many = wave_total(work.many);
    s = shared_plan_of(p.rule, work, tokens * p.g, prefix_tiles, HardwareRcp());
    int items = s.p_items;
    for (int b0 = 0; b0 < p.B; b0 += 64) {
        const int b = b0 + lane, i = min(b, p.B - 1);
        const int rows = max(tab.tok0[i + 1] - tab.tok0[i], 0) * p.g;
        const int n = b < p.B ? request_items(p.rule, s, rows, (tab.keys[i] + TK - 1) / TK, HardwareRcp()) : 0, sum = wave_sum_up(n);
        if (b < p.B) tab.items[b] = items + sum - n;
        items += __builtin_amdgcn_readlane(sum, 63);
    }
    wave_exchange();
    return items;
}

// The last b with start[b] <= x, 64 candidates at a time (start in LDS, ascending, start[0] <= x; x uniform).
__device__ __forceinline__ int last_at_most(const int* start, int count, int x) {
    const int lane = threadIdx.x & 63;
    int lo = 0, n = count;
    while (n > 1) {
        const int step = (n + 63) >> 6, i = lane * step;
        const uint64_t m = __ballot(i < n && start[min(lo + i, count - 1)] <= x);
        const int k = 63 - __builtin_clzll(m);
        lo += k * step;
        n = min(step, n - k * step);
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

// global -> LDS, 16 bytes per lane: lane l's piece lands at lds + 16 l.  Hidden from the compiler (it would drain every
// transfer in front of every LDS read); completion is awaited by hand.
__device__ __forceinline__ void dma16(unsigned lds, const char* base, unsigned off) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(lds), "v"(off), "s"(base) : "memory");
}

// One workgroup's work: rows row0 .. of a request's `rows` (or of the stacked ones), K/V head `head`, key tiles u0 .. u0 +
// n_tiles of the sequence of the prefix' tiles and the request's own.
struct SharedItem {
    int head, part, parts, before, row0, rows, u0, n_tiles, prefix_tiles, own_keys, n_tok;
    bool stacked;
    const int* own_table;
};

// Page of the 16-key group `group` of an item's range (page_of_keys; 0 from the range's end on).
template <int TK>
__device__ __forceinline__ int page_of_group(const SharedPrefixParams& p, const SharedItem& it, int group, int end) {
    constexpr int CPT = TK / 16;
    const int u = it.u0 + group / CPT, own = u - it.prefix_tiles, key = (own < 0 ? u : own) * TK + 16 * (group % CPT);
    const int keys = group >= end ? 0 : own < 0 ? p.prefix_len : it.own_keys;
    return page_of_keys(own < 0 ? p.prefix_table : it.own_table, key, keys, p.log2_page, p.n_pages);
}

// Where a row of the item lies in the workspace, once its sum of parts is known.
__device__ __forceinline__ int64_t part_slot(const SharedPrefixParams& p, const SharedItem& it, int64_t row) {
    return (int64_t)(it.before + it.part) * p.T * (p.Hkv * p.g) + row;
}

// ---------------------------------------------------------------------------------------------------------------------
// Up to 16 * RB rows: a single token's heads, or a few tokens'.  The work is bound by reading K and V, so each wave
// takes a quarter of the item's keys for itself, 16 keys (a granule, on one page) at a time, through a ring of its own:
// no barrier in the loop, and two granules and more per wave on their way (K and V through one ring of four waves with a barrier a
// tile: 3.1 TB/s where this reached 4.4; D = 256 1.4 and 4.0).  S^T = K.Q^T is one 16 x 16 block per 16 rows
// (v_mfma 16x16x32), whose registers are the B operand of O^T += V^T.P^T (16x16x16) as they are.  The four waves' sums are joined
// through LDS at the end.
// Bank conflicts: a K read takes 16 rows' 16 bytes of one column, a V read 8 rows' 32 bytes (half a wave at a time); the
// chunks of a row are exchanged so that they fall on all 64 banks.
template <typename E, int D, int RB>
__device__ __forceinline__ void shared_few_rows(const SharedPrefixParams& p, const SharedItem& it, const int (&toks)[2], char* ring) {
    using v8 = typename Elem<E>::v8;
    using v4 = typename Elem<E>::v4;
    constexpr int TK = SharedCfg<D>::kTk, CPT = TK / 16, kRow = 2 * D, kGran = 16 * kRow, CH = D / 8;
    constexpr int N = SharedCfg<D>::kStages * 2 * TK * kRow / 4 / (2 * kGran);  // granules in a wave's ring
    constexpr int NP = kGran / 1024, RPP = 1024 / kRow;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r16 = lane & 15, q4 = lane >> 4, Hq = p.Hkv * p.g, P1 = (1 << p.log2_page) - 1;
    auto k_swz = [](int row) { return CH == 8 ? (row >> 1) & 7 : row & 15; };
    auto v_swz = [](int row) { return CH == 8 ? (row & 6) : (row & 7) << 1; };

    const int all = it.n_tiles * CPT, g0 = (int)((int64_t)all * wave / 4), n = (int)((int64_t)all * (wave + 1) / 4) - g0;
    char* mine = ring + wave * N * 2 * kGran;
    const unsigned lds = __builtin_amdgcn_readfirstlane((unsigned)(size_t)(__attribute__((address_space(3))) char*)mine);
    const int d_rip = lane / CH, d_slot = lane % CH;
    unsigned k_off[NP], v_off[NP];
#pragma unroll
    for (int j = 0; j < NP; ++j) {
        const int row = RPP * j + d_rip;
        k_off[j] = (unsigned)(row * (int)p.ks.row * 2) + (unsigned)((d_slot ^ k_swz(row)) << 4);
        v_off[j] = (unsigned)(row * (int)p.vs.row * 2) + (unsigned)((d_slot ^ v_swz(row)) << 4);
    }
    const char* k_head = reinterpret_cast<const char*>(p.kc + it.head * p.ks.head);
    const char* v_head = reinterpret_cast<const char*>(p.vc + it.head * p.vs.head);
    int pages = page_of_group<TK>(p, it, g0 + lane, g0 + n), pages_next = -1;
    if (n > 64) pages_next = page_of_group<TK>(p, it, g0 + 64 + lane, g0 + n);
    int page_k = 0, row_k = 0;
    int limit[RB], hq[RB];
    v8 qf[RB][D / 32];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        const int R = min(it.row0 + 16 * rb + r16, it.rows - 1), ti = div_group(p, R);
        hq[rb] = it.head * p.g + (R - ti * p.g);
        limit[rb] = p.causal ? min(it.own_keys - 1, it.own_keys - it.n_tok + ti) : it.own_keys - 1;
        const uint16_t* qr = p.q + toks[rb] * p.q_tok + hq[rb] * p.q_head + q4 * 8;
#pragma unroll
        for (int ks = 0; ks < D / 32; ++ks) qf[rb][ks] = *reinterpret_cast<const v8*>(qr + ks * 32);
    }

    auto send_k = [&](int i) {
        if ((i & 63) == 0 && i > 0) {
            pages = pages_next;
            if (i + 64 < n) pages_next = page_of_group<TK>(p, it, g0 + i + 64 + lane, g0 + n);
        }
        const int g = g0 + i, u = it.u0 + g / CPT;
        page_k = __builtin_amdgcn_readlane(pages, i & 63);
        row_k = ((u < it.prefix_tiles ? u : u - it.prefix_tiles) * TK + 16 * (g % CPT)) & P1;
        const char* base = k_head + 2 * ((int64_t)max(page_k, 0) * p.ks.page + (int64_t)row_k * p.ks.row);
        const unsigned l = lds + (unsigned)(i % N) * 2 * kGran;
#pragma unroll
        for (int j = 0; j < NP; ++j) dma16(l + 1024u * j, base, k_off[j]);
    };
    auto send_v = [&](int i) {  // (right after send_k of the same granule, as far as pages go)
        const char* base = v_head + 2 * ((int64_t)max(page_k, 0) * p.vs.page + (int64_t)row_k * p.vs.row);
        const unsigned l = lds + (unsigned)(i % N) * 2 * kGran + kGran;
#pragma unroll
        for (int j = 0; j < NP; ++j) dma16(l + 1024u * j, base, v_off[j]);
    };
    uint64_t there = 0;  // bit j: granule i + j lies on a page
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (i < n) {
            send_k(i);
            send_v(i);
            there |= (uint64_t)(page_k >= 0) << i;
        }

    f32x4 o[RB][D / 16];
    float m_run[RB], l_run[RB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        m_run[rb] = -1e30f, l_run[rb] = 0.0f;
#pragma unroll
        for (int db = 0; db < D / 16; ++db) o[rb][db] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    int k_rd[D / 32], v_rd;
#pragma unroll
    for (int ks = 0; ks < D / 32; ++ks) k_rd[ks] = r16 * kRow + (((4 * ks + q4) ^ k_swz(r16)) << 4);
    const int v_row = 4 * q4 + (r16 >> 2);  // lane 4 q + pp of a group of 16 gives row q, 8 bytes pp
    v_rd = v_row * kRow + 8 * (lane & 1);
    const int v_ch = (lane >> 1) & 1, v_x = v_swz(v_row);
    auto v_frag = [&](const char* vb, int db) -> v4 {
        return __builtin_bit_cast(v4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                          (__attribute__((address_space(3))) short4_t*)(vb + v_rd + (((2 * db + v_ch) ^ v_x) << 4))));
    };
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)  // (waited for here: see shared_many_rows)
#pragma unroll
        for (int ks = 0; ks < D / 32; ++ks) asm volatile("" : "+v"(qf[rb][ks]));
    auto max4 = [](f32x4 s) { return max_nan(max_nan(s[0], s[1]), max_nan(s[2], s[3])); };

    int specials = 0;  // masked granules held infinities or NaN
    for (int i = 0; i < n; ++i) {
        const bool more = i + N < n;
        const char* kb = mine + (i % N) * 2 * kGran;
        const char* vb = kb + kGran;
        if (more)
            asm volatile("s_waitcnt vmcnt(%0)" : : "n"((2 * N - 1) * NP) : "memory");
        else
            wait_all_vmem();
        f32x4 s[RB];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) s[rb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int ks = 0; ks < D / 32; ++ks) {
            const v8 a = *reinterpret_cast<const v8*>(kb + k_rd[ks]);
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) s[rb] = Elem<E>::mfma16(a, qf[rb][ks], s[rb]);
        }
        if (more) {  // K's place is free: its reads have completed
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            send_k(i + N);
        }
        const int g = g0 + i, u = it.u0 + g / CPT, key = (u < it.prefix_tiles ? u : u - it.prefix_tiles) * TK + 16 * (g % CPT);
        int lim[RB];
        bool any = !(there & 1);
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            lim[rb] = (u < it.prefix_tiles ? p.prefix_len - 1 : limit[rb]) - key;
            any = any || __any(lim[rb] < 15);
        }
        const int masked = __builtin_amdgcn_readfirstlane((int)any);
        if (masked) {
#pragma unroll
            for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (4 * q4 + e > lim[rb] || !(there & 1)) s[rb][e] = -__builtin_inff();
        }
        v4 pf[RB];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            const float mx = max4(s[rb]) * p.scale_log2e;  // of this lane's four keys: the row's own is needed only when it moves
            if (!__all(mx - m_run[rb] <= kRescaleSlack)) {
                float a, b, m = mx;
                half_wave_pair(m, a, b);
                m = max_nan(a, b);
                m = max_nan(m, __shfl_xor(m, 16));
                const float m_new = max_nan(m_run[rb], m), alpha = __builtin_amdgcn_exp2f(m_run[rb] - m_new);
                m_run[rb] = m_new;
                l_run[rb] *= alpha;
#pragma unroll
                for (int db = 0; db < D / 16; ++db)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[rb][db][e] *= alpha;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[rb][e], p.scale_log2e, -m_run[rb]));
                l_run[rb] += x;
                pf[rb][e] = (E)x;
            }
        }
        if (more)
            asm volatile("s_waitcnt vmcnt(%0)" : : "n"((2 * N - 1) * NP) : "memory");
        if (!masked) {
#pragma unroll
            for (int db = 0; db < D / 16; ++db) {
                const v4 a = v_frag(vb, db);
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) o[rb][db] = Elem<E>::mfma16(a, pf[rb], o[rb][db]);
            }
        } else {
            bool special = false;
#pragma unroll
            for (int db = 0; db < D / 16; ++db) {
                const v4 a = finite_part<E>(v_frag(vb, db), special);
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) o[rb][db] = Elem<E>::mfma16(a, pf[rb], o[rb][db]);
            }
            specials |= __builtin_amdgcn_readfirstlane((int)__any(special));
        }
        there >>= 1;
        if (more) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            send_v(i + N);
            there |= (uint64_t)(page_k >= 0) << (N - 1);
        }
    }
    wait_all_vmem();
    if (__builtin_expect(specials != 0, 0)) {
        // the values taken out of masked granules, to the rows that do see them: those granules once more, one at a time
#pragma unroll 1
        for (int i = 0; i < n; ++i) {
            const int g = g0 + i, u = it.u0 + g / CPT, key = (u < it.prefix_tiles ? u : u - it.prefix_tiles) * TK + 16 * (g % CPT);
            const int page = __builtin_amdgcn_readfirstlane(page_of_group<TK>(p, it, g, g0 + n));
            const int pre = u < it.prefix_tiles;
            bool any = false;
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) any = any || __any((pre ? p.prefix_len - 1 : limit[rb]) - key < 15);
            if (page < 0 || !any) continue;
            const char* base = v_head + 2 * ((int64_t)page * p.vs.page + (int64_t)(key & P1) * p.vs.row);
#pragma unroll
            for (int j = 0; j < NP; ++j) dma16(lds + 1024u * j, base, v_off[j]);
            wait_all_vmem();
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                v4 sees;
#pragma unroll
                for (int e = 0; e < 4; ++e) sees[e] = (E)(4 * q4 + e <= (pre ? p.prefix_len - 1 : limit[rb]) - key ? 1.0f : 0.0f);
#pragma unroll
                for (int db = 0; db < D / 16; ++db) {
                    const v4 f = v_frag(mine, db);
#pragma unroll
                    for (int kind = 1; kind <= 3; ++kind) {
                        const f32x4 c = Elem<E>::mfma16(special_part<E>(f, kind), sees, f32x4{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[rb][db][e] += c[e] > 0.0f ? special_value(kind) : 0.0f;
                    }
                }
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
    }

    // ---- the four waves' sums: 16 rows at a time through LDS, rows padded so that a store's 16 rows fall on all banks
    constexpr int kOut = D + 4;  // floats
    float* lo = reinterpret_cast<float*>(ring);
    float* lml = lo + 4 * 16 * kOut;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        float a, b;
        half_wave_pair(l_run[rb], a, b);
        float l = a + b;
        l += __shfl_xor(l, 16);
        __syncthreads();  // (every wave is done with its ring, or with the rows before)
        if (q4 == 0) {
            lml[(wave * 16 + r16) * 2] = m_run[rb];
            lml[(wave * 16 + r16) * 2 + 1] = l;
        }
#pragma unroll
        for (int db = 0; db < D / 16; ++db) *reinterpret_cast<f32x4*>(lo + (wave * 16 + r16) * kOut + 16 * db + 4 * q4) = o[rb][db];
        int* where = reinterpret_cast<int*>(lml + 128);  // token and head of each row
        if (wave == 0 && q4 == 0) {
            where[2 * r16] = toks[rb];
            where[2 * r16 + 1] = hq[rb];
        }
        __syncthreads();
        constexpr int C4 = D / 4;
        for (int x = tid; x < 16 * C4; x += 256) {
            const int row = x / C4, c = x % C4;
            if (it.row0 + 16 * rb + row >= it.rows) continue;
            float m = -1e30f, sum = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; ++w) m = max_nan(m, lml[(w * 16 + row) * 2]);
            f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float f = __builtin_amdgcn_exp2f(lml[(w * 16 + row) * 2] - m);
                sum += f * lml[(w * 16 + row) * 2 + 1];
                acc += *reinterpret_cast<const f32x4*>(lo + (w * 16 + row) * kOut + 4 * c) * f;
            }
            const int tok = where[2 * row], h = where[2 * row + 1];
            const int64_t at = (int64_t)tok * Hq + h;
            const int total = it.before + it.parts;
            if (!it.stacked && it.part == 0 && c == 0) p.row_parts[at] = total == 1 ? 0 : total;
            if (!it.stacked && total == 1) {
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                v4 y;
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = (E)(acc[e] * inv);
                *reinterpret_cast<v4*>(p.o + tok * p.o_tok + h * p.o_head + 4 * c) = y;
            } else {
                const int64_t slot = part_slot(p, it, at);
                if (c == 0) *reinterpret_cast<f32x2*>(p.part_ml + 2 * slot) = f32x2{m, sum};
                *reinterpret_cast<f32x4*>(p.part_o + slot * D + 4 * c) = acc;
            }
        }
    }
}

// Many rows: four waves of 32, key tiles of kTk keys shared through a ring of four stages (three on their way), one barrier a
// tile.  Scores of tile t + 1 run on the matrix pipe beside the exponentials of tile t, then V^T.P^T beside the maximum of t + 1,
// written out instruction by instruction; O lies in named accumulator registers, which the compiler neither copies nor
// counts.  That interleaving took one prompt of 4 096 tokens behind 8 192 keys (D = 128) from 760 to 913 TFLOP/s, less scalar work
// to 954, transfers in pairs and Q's loads beside the first pages' to 1 006 (966 - 1 017 on other boxes).
// What bounds it (counters of that prompt, profiles/paged_counters.txt): the matrix pipe is busy 48 % of the time (D = 256, 16
// heads on 4: 45 %); of the waves' cycles 32 % (17 %) wait to issue and 22 % (28 %) for memory, LDS or the barrier.  A plain
// instruction takes 4.7 cycles, an exponential 8.7, a matrix instruction 32, and a step of D = 128 has 69 vector instructions to 16
// matrix ones; two waves share a SIMD at D = 64 and 128 (183 + 32 and 154 + 64 registers), one has it at D = 256.  How much of the
// rest is the barrier of each tile, the wait between scores and V, or the masked tiles was not separated.  64 rows to a
// wave would halve the LDS reads and the transfers; built, it ran at 940 where this ran at 979 (two waves to a workgroup), and
// needed more registers than there are where its other costs were cut.
template <typename E, int D>
__device__ __forceinline__ void shared_many_rows(const SharedPrefixParams& p, const SharedItem& it, int tok, char* ring) {
    using HD = HeadDim<D>;
    using CFG = SharedCfg<D>;
    using v8 = typename Elem<E>::v8;
    constexpr int TK = CFG::kTk, KB = TK / 32, ST = CFG::kStages, kTile = TK * HD::kRow, kStage = 2 * kTile;
    constexpr int PPW = kTile / 1024 / 4;            // 1 KiB pieces of a K (or V) tile that each wave moves
    constexpr int RPP = 1024 / HD::kRow;             // rows per piece
    constexpr int RPW = RPP * PPW;                   // rows per wave and tile: 16 (D = 64) or 8, on one page
    constexpr int CPT = TK / 16;                     // 16-key groups per tile
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const LaneGeomD<D> geo = make_lane_geom_d<D>(lane);
    const int P1 = (1 << p.log2_page) - 1;  // (row in a page)
    const int R_off = wave * 32 + geo.r, head = it.head, row0 = it.row0, rows = it.rows, u0 = it.u0, n_tiles = it.n_tiles;
    const bool valid = row0 + R_off < rows, wave_valid = row0 + wave * 32 < rows;
    const int R = min(row0 + R_off, rows - 1), ti = div_group(p, R), hq = head * p.g + (R - ti * p.g), Hq = p.Hkv * p.g;
    const int own_limit = p.causal ? min(it.own_keys - 1, it.own_keys - it.n_tok + ti) : it.own_keys - 1;  // the last own key this row sees

    // ---- transfers: this wave moves rows RPW * wave .. of each tile, which lie on one page.  Lane L holds where the 16-key
    //      group L of a run of 64 begins in K and in V (bytes from the head's first row; page 0 for a group on no page: its
    //      scores are masked); the next run's pages are on their way meanwhile.  Lane l fills slot l % kChunks of row
    //      l / kChunks of a piece with the chunk the swizzle maps there; the instruction's offset moves both sides, so it is taken
    //      off the source's (rows are at least D apart: what remains is not negative).
    const unsigned ring_lds = __builtin_amdgcn_readfirstlane((unsigned)(size_t)(__attribute__((address_space(3))) char*)ring);
    const int d_rip = lane / HD::kChunks, d_slot = lane % HD::kChunks, kr = 2 * (int)p.ks.row, vr = 2 * (int)p.vs.row;
    unsigned k_off[PPW], v_off[PPW];
#pragma unroll
    for (int j = 0; j < PPW; ++j) {
        const int row = RPW * wave + RPP * j + d_rip;
        k_off[j] = (unsigned)((RPP * j + d_rip) * kr) + (unsigned)((d_slot ^ (row & HD::kKMask)) << 4) - 1024u * j;
        v_off[j] = (unsigned)((RPP * j + d_rip) * vr) + (unsigned)((d_slot ^ ((row & HD::kVMask) << 2)) << 4) - 1024u * j;
    }
    const char* k_head = reinterpret_cast<const char*>(p.kc + head * p.ks.head) + (RPW * wave % 16) * (int64_t)kr;
    const char* v_head = reinterpret_cast<const char*>(p.vc + head * p.vs.head) + (RPW * wave % 16) * (int64_t)vr;
    const int n_groups = n_tiles * CPT;
    auto load_pages = [&](int group) -> int { return page_of_group<TK>(p, it, group + lane, n_groups); };
    int pages_next = load_pages(0);
    // Lane L: whether group L of the run of 64 lies on no page (bit 0), of the run before (bit 1), of any run so far (bit 2).  Tiles
    // near such a group take the masked form, by the one number that the steps look at.
    int pageless = 0, near_pageless = 0;
    // (Q's loads go out beside the first pages')
    v8 qf[HD::kSteps];
    {
        const uint16_t* qr = p.q + tok * p.q_tok + hq * p.q_head + geo.hh * 8;
#pragma unroll
        for (int ks = 0; ks < HD::kSteps; ++ks) qf[ks] = *reinterpret_cast<const v8*>(qr + ks * 16);
    }

    uint64_t k_at = 0, v_at = 0;
    auto refill = [&](int g0) {
        const int page = max(pages_next, 0), u = u0 + (g0 + lane) / CPT;
        const int row = ((u < it.prefix_tiles ? u : u - it.prefix_tiles) * TK + 16 * (lane % CPT)) & P1;
        pageless = (pageless & 4) | (pageless & 1) << 1 | (pages_next < 0 && g0 + lane < n_groups ? 5 : 0);
        near_pageless = __builtin_amdgcn_readfirstlane((int)__any(pageless & 3));
        k_at = 2 * ((int64_t)page * p.ks.page + (int64_t)row * p.ks.row);
        v_at = 2 * ((int64_t)page * p.vs.page + (int64_t)row * p.vs.row);
        if (g0 + 64 < n_groups) pages_next = load_pages(g0 + 64);
    };
    struct Transfer {
        const char *k, *v;
        unsigned lds;
    };
    auto lane64 = [](uint64_t x, int l) -> uint64_t {
        const unsigned lo = __builtin_amdgcn_readlane((unsigned)x, l), hi = __builtin_amdgcn_readlane((unsigned)(x >> 32), l);
        return (uint64_t)hi << 32 | lo;
    };
    auto transfer = [&](int t) -> Transfer {
        const int g0 = t * CPT;
        if ((g0 & 63) == 0) refill(g0);
        const int l = (g0 + RPW * wave / 16) & 63;
        return {k_head + lane64(k_at, l), v_head + lane64(v_at, l), ring_lds + (unsigned)(t % ST) * kStage + (unsigned)(PPW * wave) * 1024u};
    };
    // Two pieces of K (first half of the indices) or of V in one go.  on > 0: all lanes, else none (a step past the last transfer
    // issues its pieces too, for the count that is waited for).
    auto send_pair = [&](const Transfer& tr, int on, auto jc) {
        constexpr int j = 2 * decltype(jc)::value % PPW;
        constexpr bool val = 2 * decltype(jc)::value >= PPW;
        const unsigned lds = tr.lds + (val ? kTile : 0), off0 = val ? v_off[j] : k_off[j], off1 = val ? v_off[j + 1] : k_off[j + 1];
        const char* base = val ? tr.v : tr.k;
        asm volatile(
            "s_cmp_gt_i32 %6, 0\n\ts_cselect_b64 exec, -1, 0\n\ts_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %3 offset:%4\n\t"
            "global_load_lds_dwordx4 %2, %3 offset:%5\n\ts_mov_b64 exec, -1"
            :
            : "s"(lds), "v"(off0), "v"(off1), "s"(base), "n"(1024 * j), "n"(1024 * (j + 1)), "s"(on)
            : "memory", "scc");
    };
#pragma unroll
    for (int t = 0; t < ST - 1; ++t)
        if (t < n_tiles) {
            const Transfer tr = transfer(t);
            static_for<PPW>([&](auto ic) { send_pair(tr, 1, ic); });
        }

    f32x16 s_cur[KB], s_next[KB];
    float m_run = -1e30f, l_run = 0.0f;
    const float c = p.scale_log2e;

    auto k_frag = [&](const char* kb, int i) -> v8 { return *reinterpret_cast<const v8*>(kb + geo.k_rd[i / KB] + (i % KB) * 32 * HD::kRow); };
    auto v_frag = [&](const char* vb, int kk, int db) -> v8 {
        const char* a0 = vb + geo.v_rd[db] + kk * 16 * HD::kRow;
        const short4_t t0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t*)(a0));
        const short4_t t1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t*)(a0 + 8 * HD::kRow));
        return __builtin_bit_cast(v8, __builtin_shufflevector(t0, t1, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    // the last key of tile t that the row sees, counted from the tile's first; whether the tile needs the mask
    auto limit_of = [&](int t) -> int {
        const int u = u0 + t, own = u - it.prefix_tiles;
        return (own < 0 ? p.prefix_len - 1 : own_limit) - (own < 0 ? u : own) * TK;
    };
    // tiles that need no mask for any row of the wave: all but the one that the prefix' end cuts and those from the first one
    // that some row's limit cuts on
    int own_from;
    {
        int low = own_limit;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) low = min(low, __shfl_xor(low, d));
        own_from = it.prefix_tiles - u0 + (__builtin_amdgcn_readfirstlane(low) + 1) / TK;
    }
    const int cut = p.prefix_len % TK != 0 ? it.prefix_tiles - 1 - u0 : -1;
    auto needs_mask = [&](int t) -> int { return (int)(t >= own_from) | (int)(t == cut) | near_pageless; };
    // the groups of tile t that lie on a page; looked at when the transfers have reached tile t + ST - 2
    auto groups_of = [&](int t) -> unsigned {
        return ((1u << CPT) - 1) & ~pageless_groups(__ballot((pageless & 2) != 0), __ballot((pageless & 1) != 0), t, ST - 2, CPT);
    };
    auto mask_scores = [&](f32x16 (&s)[KB], int lim, unsigned groups) {
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int k = 32 * b + 8 * (e >> 2) + (e & 3);
                if (k + 4 * geo.hh > lim || !((groups >> (k >> 4)) & 1)) s[b][e] = -__builtin_inff();
            }
    };
    auto lane_max = [&](const f32x16 (&s)[KB]) -> float {
        float m = max_nan(s[0][0], s[0][1]);
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int e = b == 0 ? 2 : 0; e < 16; e += 2) m = max_nan(max_nan(m, s[b][e]), s[b][e + 1]);
        return m * c;
    };
    // the reference moves only when some row's score passes it by more than kRescaleSlack: this lane's half of the tile's keys
    // decides, the two halves meet only then
    auto rescale = [&](float mx) {
        if (__builtin_expect(__all(mx - m_run <= kRescaleSlack), 1)) return;
        float a, b;
        half_wave_pair(mx, a, b);
        const float m_new = max_nan(m_run, max_nan(a, b)), alpha = __builtin_amdgcn_exp2f(m_run - m_new);
        m_run = m_new;
        l_run *= alpha;
        acc_scale_n<0, 16 * HD::kBlocks>(alpha);
    };

    constexpr int NS = HD::kSteps * KB, NE = 16 * KB, NV = 2 * KB * HD::kBlocks, AHEAD = 4;
    int specials = 0;  // masked tiles held infinities or NaN in V
    int masked = 0;  // (whole numbers in scalar registers: a branch on a lane mask would keep both sides' registers alive)
    // Q is waited for HERE: left pending, the waits in front of its uses would drain the loop's transfers
#pragma unroll
    for (int ks = 0; ks < HD::kSteps; ++ks) asm volatile("" : "+v"(qf[ks]));
    wait_all_vmem();
    __syncthreads();
    if constexpr (D == 64)
        acc_reserve32();
    else if constexpr (D == 128)
        acc_reserve64();
    else
        acc_reserve128();
    static_for<HD::kBlocks>([&](auto ic) { acc_zero16<16 * decltype(ic)::value>(); });
    if (wave_valid && n_tiles > 0) {
        masked = needs_mask(0);
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e) s_cur[b][e] = 0.0f;
#pragma unroll
        for (int i = 0; i < NS; ++i) s_cur[i % KB] = Elem<E>::mfma(k_frag(ring, i), qf[i / KB], s_cur[i % KB]);
        if (masked) mask_scores(s_cur, limit_of(0), groups_of(0));
        rescale(lane_max(s_cur));
    }
    // Step t: while the matrix pipe computes the next tile's scores, the vector ALU turns this tile's into probabilities; while
    // it multiplies those with V, the vector ALU takes the next scores' maximum.  Written out gap by gap: one MFMA, that
    // gap's share of the vector work, the operand read AHEAD MFMAs later, one piece of the step's transfer.
    auto step = [&](int t, auto stage) {
        constexpr int S = decltype(stage)::value;  // t % ST, so that the LDS reads' offsets are constants
        const bool more = t + 1 < n_tiles;
        const int on = n_tiles - (t + ST - 1);  // > 0: tile t + ST - 1, into the stage of tile t - 1, which every wave has left
        const Transfer tr = transfer(t + ST - 1);
        if (wave_valid) {
            const char* kb = ring + (S + 1) % ST * kStage;
            const char* vb = ring + S * kStage + kTile;
            v8 pf[2 * KB], kf[AHEAD], vf[AHEAD];
            float sum = 0.0f;
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
                for (int e = 0; e < 16; ++e) s_next[b][e] = 0.0f;
            // (past the last tile the scores of whatever the stage holds: never used)
            static_for<AHEAD>([&](auto ic) { kf[decltype(ic)::value] = k_frag(kb, decltype(ic)::value); });
            static_for<NS>([&](auto ic) {
                constexpr int i = decltype(ic)::value;
                s_next[i % KB] = Elem<E>::mfma(kf[i % AHEAD], qf[i / KB], s_next[i % KB]);
                if constexpr (i + AHEAD < NS) kf[i % AHEAD] = k_frag(kb, i + AHEAD);
                constexpr int every = NS / PPW;
                if constexpr (i % every == every - 1) send_pair(tr, on, std::integral_constant<int, i / every>{});
                static_for<NE / NS>([&](auto jc) {
                    constexpr int e = i * (NE / NS) + decltype(jc)::value;
                    const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s_cur[e / 16][e % 16], c, -m_run));
                    s_cur[e / 16][e % 16] = x;
                    if constexpr (e > 0) sum += s_cur[(e - 1) / 16][(e - 1) % 16];
                    if constexpr (e % 2 == 1 && e >= 3) {
                        pf[(e - 3) / 8][(e - 3) % 8] = (E)s_cur[(e - 3) / 16][(e - 3) % 16];
                        pf[(e - 2) / 8][(e - 2) % 8] = (E)s_cur[(e - 2) / 16][(e - 2) % 16];
                    }
                });
                __builtin_amdgcn_sched_barrier(0);
            });
            sum += s_cur[KB - 1][15];
            l_run += sum;
            pf[2 * KB - 1][6] = (E)s_cur[KB - 1][14];
            pf[2 * KB - 1][7] = (E)s_cur[KB - 1][15];
            // (pinned here: left alone the compiler sinks the vector work into the block that uses it)
#pragma unroll
            for (int j = 0; j < 2 * KB; ++j) asm volatile("" : "+v"(pf[j]));
            asm volatile("s_nop 4" : "+v"(l_run));  // (wait states between a vector write and the MFMAs that read it)

            const int masked_next = needs_mask(t + 1);
            if (__builtin_expect(masked_next != 0, 0)) mask_scores(s_next, limit_of(t + 1), groups_of(t + 1));
            float mx;
            if (__builtin_expect(masked == 0, 1)) {
                static_for<AHEAD>([&](auto ic) { vf[decltype(ic)::value] = v_frag(vb, decltype(ic)::value / HD::kBlocks, decltype(ic)::value % HD::kBlocks); });
                mx = max_nan(s_next[0][0], s_next[0][1]);
                static_for<NV>([&](auto ic) {
                    constexpr int i = decltype(ic)::value;
                    Elem<E>::template mfma_owned<16 * (i % HD::kBlocks)>(vf[i % AHEAD], pf[i / HD::kBlocks]);
                    if constexpr (i + AHEAD < NV) vf[i % AHEAD] = v_frag(vb, (i + AHEAD) / HD::kBlocks, (i + AHEAD) % HD::kBlocks);
                    if constexpr (i >= 2) {  // links of the maximum, from the third gap on
                        constexpr int NL = 8 * KB - 1, lo = (i - 2) * NL / (NV - 2), hi = (i - 1) * NL / (NV - 2);
                        static_for<hi - lo>([&](auto jc) {
                            constexpr int e = 2 * (lo + decltype(jc)::value + 1);
                            mx = max_nan(max_nan(mx, s_next[e / 16][e % 16]), s_next[e / 16][e % 16 + 1]);
                        });
                    }
                    __builtin_amdgcn_sched_barrier(0);
                });
                mx *= c;
            } else {
                bool special = false;
                static_for<NV>([&](auto ic) {
                    constexpr int kk = decltype(ic)::value / HD::kBlocks, db = decltype(ic)::value % HD::kBlocks;
                    v8 f = finite_part<E>(v_frag(vb, kk, db), special);
                    asm volatile("s_nop 4" : "+v"(f));
                    Elem<E>::template mfma_owned<16 * db>(f, pf[kk]);
                });
                specials |= __builtin_amdgcn_readfirstlane((int)__any(special));
                mx = lane_max(s_next);
            }
            if (more) {
                rescale(mx);
                masked = masked_next;
#pragma unroll
                for (int b = 0; b < KB; ++b) s_cur[b] = s_next[b];
            }
        } else {
            static_for<PPW>([&](auto ic) { send_pair(tr, on, ic); });
        }
        // this wave's share of tile t + 2 has landed (transfers complete in order); what was sent since stays in flight
        asm volatile("s_waitcnt vmcnt(%0)" : : "n"((ST - 3) * 2 * PPW) : "memory");
        __syncthreads();
    };
    for (int t = 0; t < n_tiles;) {
        step(t, std::integral_constant<int, 0>{});
        if (++t == n_tiles) break;
        step(t, std::integral_constant<int, 1>{});
        if (++t == n_tiles) break;
        step(t, std::integral_constant<int, 2>{});
        if (++t == n_tiles) break;
        step(t, std::integral_constant<int, 3>{});
        ++t;
    }

    acc_fence();
    if (__builtin_expect(specials != 0, 0)) {
        // the values taken out of masked tiles, to the rows that do see them: those tiles' V once more, in the quarter of the
        // ring that is this wave's own now
        const int had_pageless = __builtin_amdgcn_readfirstlane((int)__any(pageless & 4));
        char* mine = ring + wave * (ST * kStage / 4);
        const unsigned mine_lds = ring_lds + (unsigned)(wave * (ST * kStage / 4));
#pragma unroll 1
        for (int t = 0; t < n_tiles; ++t) {
            const int u = u0 + t, key = (u < it.prefix_tiles ? u : u - it.prefix_tiles) * TK, lim = limit_of(t);
            if (!(needs_mask(t) | had_pageless)) continue;  // (the other tiles' were multiplied as they are)
            unsigned groups = (1u << CPT) - 1;
            if (had_pageless)
#pragma unroll 1
                for (int g = 0; g < CPT; ++g)
                    if (__builtin_amdgcn_readfirstlane(page_of_group<TK>(p, it, t * CPT + g, n_groups)) < 0) groups &= ~(1u << g);
            const char* v_rows = reinterpret_cast<const char*>(p.vc + head * p.vs.head);
#pragma unroll 1
            for (int j = 0; j < kTile / 1024; ++j) {
                const int row = RPP * j, page = __builtin_amdgcn_readfirstlane(page_of_group<TK>(p, it, t * CPT + row / 16, n_groups));
                const char* vb = v_rows + 2 * ((int64_t)max(page, 0) * p.vs.page + (int64_t)((key + row) & P1) * p.vs.row);
                dma16(mine_lds + 1024u * j, vb, (unsigned)(d_rip * (int)p.vs.row * 2) + (unsigned)((d_slot ^ (((row + d_rip) & HD::kVMask) << 2)) << 4));
            }
            wait_all_vmem();
            v8 sees[2 * KB];  // 1 where the row sees the key
#pragma unroll
            for (int kk = 0; kk < 2 * KB; ++kk)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int k = 16 * kk + 8 * (i >> 2) + (i & 3);
                    sees[kk][i] = (E)(k + 4 * geo.hh <= lim && ((groups >> (k >> 4)) & 1) ? 1.0f : 0.0f);
                }
            static_for<HD::kBlocks>([&](auto dc) {
                constexpr int db = decltype(dc)::value;
#pragma unroll 1
                for (int kind = 1; kind <= 3; ++kind) {
                    f32x16 n;
#pragma unroll
                    for (int e = 0; e < 16; ++e) n[e] = 0.0f;
#pragma unroll
                    for (int kk = 0; kk < 2 * KB; ++kk) n = Elem<E>::mfma(special_part<E>(v_frag(mine, kk, db), kind), sees[kk], n);
                    static_for<16>([&](auto ec) {
                        constexpr int e = decltype(ec)::value;
                        const float x = acc_get<16 * db + e>();
                        acc_put<16 * db + e>(n[e] > 0.0f ? x + special_value(kind) : x);
                    });
                }
            });
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
    }

    // ---- out: whole rows, through the quarter of the ring that is this wave's own now (stored from the accumulator's layout a
    //      wave instruction would touch 32 rows with 32 bytes each); chunk c of row r lies at c ^ (r & 15)
    float l0, l1;
    half_wave_pair(l_run, l0, l1);
    const float l = l0 + l1;
    const int total = it.before + it.parts, row = tok * Hq + hq;
    const bool direct = !it.stacked && total == 1;
    if (valid && geo.hh == 0) {
        if (!it.stacked && it.part == 0) p.row_parts[row] = direct ? 0 : total;
        if (!direct) *reinterpret_cast<f32x2*>(p.part_ml + 2 * part_slot(p, it, row)) = f32x2{m_run, l};
    }
    if (!wave_valid || (n_tiles == 0 && !direct)) return;  // (nothing is read of a part whose sum is 0)
    const float scale = !direct ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
    char* st = ring + wave * (ST * kStage / 4);
    if (direct) {
        constexpr int CH = D / 8;  // 16-byte chunks of an output row
        static_for<HD::kBlocks * 4>([&](auto ic) {
            constexpr int i = decltype(ic)::value;
            const typename Elem<E>::v4 x = {(E)(acc_get<4 * i>() * scale), (E)(acc_get<4 * i + 1>() * scale), (E)(acc_get<4 * i + 2>() * scale),
                                            (E)(acc_get<4 * i + 3>() * scale)};
            *reinterpret_cast<u32x2*>(st + geo.r * 2 * D + ((i ^ (geo.r & (CH - 1) & 15)) << 4) + 8 * geo.hh) = __builtin_bit_cast(u32x2, x);
        });
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int i = 0; i < CH / 2; ++i) {
            const int r = i * (64 / CH) + lane / CH, c = lane % CH, tk = __shfl(tok, r), h = __shfl(hq, r);
            const u32x4 x = *reinterpret_cast<const u32x4*>(st + r * 2 * D + ((c ^ (r & (CH - 1) & 15)) << 4));
            if (row0 + wave * 32 + r < rows) *reinterpret_cast<u32x4*>(p.o + tk * p.o_tok + h * p.o_head + 8 * c) = x;
        }
        return;
    }
    constexpr int CH = D / 4;  // 16-byte chunks of a row of the state
    static_for<HD::kBlocks * 4>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        *reinterpret_cast<f32x4*>(st + geo.r * 4 * D + (((2 * i + geo.hh) ^ (geo.r & 15)) << 4)) =
            f32x4{acc_get<4 * i>(), acc_get<4 * i + 1>(), acc_get<4 * i + 2>(), acc_get<4 * i + 3>()};
    });
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    float* po = p.part_o + part_slot(p, it, 0) * D;
#pragma unroll 4
    for (int i = 0; i < CH / 2; ++i) {
        const int r = i * (64 / CH) + lane / CH, c = lane % CH, rw = __shfl(row, r);
        const f32x4 x = *reinterpret_cast<const f32x4*>(st + r * 4 * D + ((c ^ (r & 15)) << 4));
        if (row0 + wave * 32 + r < rows) *reinterpret_cast<f32x4*>(po + (int64_t)rw * D + 4 * c) = x;
    }
}

template <typename E, int D>
__device__ __forceinline__ void shared_prefix_body(const SharedPrefixParams& p) {
    using CFG = SharedCfg<D>;
    constexpr int TK = CFG::kTk;
    __shared__ __attribute__((aligned(1024))) char ring[SharedCfg<D>::kStages * 2 * TK * 2 * D];
    SharedItem it;
    int toks[2];  // of this lane's rows: 32 wave + (lane & 31), or, of few rows, (lane & 15) and 16 + (lane & 15)
    bool few;
    {
        const SharedTables tab(ring, p.B);  // (free until the first transfer)
        SharedPlan plan;
        const int x = (int)blockIdx.x, lane = threadIdx.x & 63;
        if (x >= shared_plan<TK>(p, plan, tab)) return;
        it.prefix_tiles = plan.prefix_tiles;
        it.stacked = x < plan.p_items;
        int unit, tile, tiles, tok0 = 0, first_item = 0;
        it.own_keys = it.n_tok = 0;
        it.own_table = nullptr;
        if (it.stacked) {
            it.rows = plan.stacked, it.parts = plan.prefix_parts, tiles = tiles_of(p.rule, plan.stacked);
        } else {
            const int b = last_at_most(tab.items, p.B, x);
            tok0 = __builtin_amdgcn_readfirstlane(tab.tok0[b]);
            it.n_tok = max(__builtin_amdgcn_readfirstlane(tab.tok0[b + 1]) - tok0, 0);
            it.own_keys = __builtin_amdgcn_readfirstlane(tab.keys[b]);
            first_item = __builtin_amdgcn_readfirstlane(tab.items[b]);
            it.rows = it.n_tok * p.g;
            tiles = tiles_of(p.rule, it.rows);
            it.parts = __builtin_amdgcn_readfirstlane(request_parts(p.rule, plan, it.rows, (it.own_keys + TK - 1) / TK, HardwareRcp()));
            it.own_table = p.block_table + b * p.table_stride;
        }
        unit_and_tile(x - first_item, p.Hkv * it.parts, tiles, unit, tile, HardwareRcp());
        unit = __builtin_amdgcn_readfirstlane(unit), tile = __builtin_amdgcn_readfirstlane(tile);
        it.head = __builtin_amdgcn_readfirstlane(quick_div(unit, it.parts, HardwareRcp())), it.part = unit - it.head * it.parts, it.row0 = tile * tile_rows(p.rule, it.rows);
        // the key tiles of this row tile: no row of it sees further than its last one
        const int end = min(it.row0 + tile_rows(p.rule, it.rows), it.rows);
        const int see = p.causal ? min(it.own_keys, it.own_keys - it.n_tok + div_group(p, end - 1) + 1) : it.own_keys;
        const int first = it.stacked || it.rows >= kRowTile ? 0 : plan.prefix_tiles;
        const int last = it.stacked ? plan.prefix_tiles : plan.prefix_tiles + (max(see, 0) + TK - 1) / TK;
        it.before = first > 0 ? plan.prefix_parts : 0;  // (parts that P items add in front of this item's)
        range_of(first, last, it.part, it.parts, it.u0, it.n_tiles, HardwareRcp());
        // (the same in every lane, though some came through the vector ALU)
        it.parts = __builtin_amdgcn_readfirstlane(it.parts), it.part = __builtin_amdgcn_readfirstlane(it.part);
        it.before = __builtin_amdgcn_readfirstlane(it.before), it.rows = __builtin_amdgcn_readfirstlane(it.rows);
        it.u0 = __builtin_amdgcn_readfirstlane(it.u0), it.n_tiles = __builtin_amdgcn_readfirstlane(it.n_tiles);
        few = it.rows <= p.rule.few_rows;
        auto token = [&](int off) -> int {
            const int t = div_group(p, min(it.row0 + off, it.rows - 1));
            if (!it.stacked) return tok0 + t;
            const int o = owner_of(tab.stacked, p.B, t);
            return tab.tok0[o] + t - tab.stacked[o];
        };
        toks[0] = token(few ? lane & 15 : (int)(threadIdx.x >> 6) * 32 + (lane & 31));
        toks[1] = few && CFG::kFewBlocks > 1 ? token(16 + (lane & 15)) : toks[0];
        __syncthreads();  // (the tables above have been read)
    }
    if (!few)
        shared_many_rows<E, D>(p, it, toks[0], ring);
    else if (CFG::kFewBlocks == 1 || it.rows - it.row0 <= 16)
        shared_few_rows<E, D, 1>(p, it, toks, ring);
    else
        shared_few_rows<E, D, CFG::kFewBlocks>(p, it, toks, ring);
}

// Two workgroups share a compute unit (D = 64, 128): architectural and accumulator registers together within 256.  The
// compiler halves that between the two kinds when asked for two; it is asked for one, with the architectural count given.
#define FA_SHARED_KERNEL(name, E, D, VGPRS) \
    __global__ __launch_bounds__(256, 1) __attribute__((amdgpu_num_vgpr(VGPRS))) void name(const SharedPrefixParams p) { shared_prefix_body<E, D>(p); }
FA_SHARED_KERNEL(fa_shared_prefix_f16_d64_kernel, _Float16, 64, 224)
FA_SHARED_KERNEL(fa_shared_prefix_f16_d128_kernel, _Float16, 128, 192)
FA_SHARED_KERNEL(fa_shared_prefix_f16_d256_kernel, _Float16, 256, 256)
FA_SHARED_KERNEL(fa_shared_prefix_bf16_d64_kernel, __bf16, 64, 224)
FA_SHARED_KERNEL(fa_shared_prefix_bf16_d128_kernel, __bf16, 128, 192)
FA_SHARED_KERNEL(fa_shared_prefix_bf16_d256_kernel, __bf16, 256, 256)
#undef FA_SHARED_KERNEL

// O = sum_s w_s o_s / sum_s w_s l_s,  w_s = exp2(m_s - max_s m_s): D / 4 lanes per row, four parts in flight.  Rows of no
// request and rows that are written already are left alone.  Bound by latency and by the bytes of the parts (a row of D floats
// each, out of the last-level cache as a rule): four parts at a time; 32 requests of 32 heads at D = 128 5.6 us, 128 of 64 heads 8.1.
template <typename E, int D>
__global__ __launch_bounds__(256) void fa_shared_prefix_merge_kernel(const SharedPrefixParams p) {
    constexpr int LPR = D / 4, RPB = 256 / LPR, U = 4;
    const int c = threadIdx.x % LPR, Hq = p.Hkv * p.g;
    const int64_t rows = (int64_t)p.T * Hq, i = (int64_t)blockIdx.x * RPB + threadIdx.x / LPR;
    if (i >= rows) return;
    const int tok = (int)(i / Hq), hq = (int)(i - (int64_t)tok * Hq);
    const int first = p.q_start[0], last = p.q_start[p.B], parts = min(p.row_parts[i], p.rule.max_prefix_parts + p.rule.max_own_parts);
    if (tok < first || tok >= last || parts <= 0) return;
    const f32x2* ml = reinterpret_cast<const f32x2*>(p.part_ml) + i;
    const float* po = p.part_o + i * D + 4 * c;
    float m = -1e30f, l = 0.0f;
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s0 = 0; s0 < parts; s0 += U) {
        f32x2 x[U];
        f32x4 o[U];
#pragma unroll
        for (int s = 0; s < U; ++s) x[s] = ml[min(s0 + s, parts - 1) * rows];
#pragma unroll
        for (int s = 0; s < U; ++s) o[s] = *reinterpret_cast<const f32x4*>(po + min(s0 + s, parts - 1) * rows * D);
        float mx = m;
#pragma unroll
        for (int s = 0; s < U; ++s) mx = max_nan(mx, x[s][0]);
        const float a = __builtin_amdgcn_exp2f(m - mx);
        m = mx, l *= a, acc *= a;
#pragma unroll
        for (int s = 0; s < U; ++s) {
            const bool there = s0 + s < parts && x[s][1] != 0.0f;
            const float w = there ? __builtin_amdgcn_exp2f(x[s][0] - m) : 0.0f;
            l += w * x[s][1];
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] += there ? w * o[s][e] : 0.0f;
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    typename Elem<E>::v4 out;
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] = (E)(acc[e] * inv);
    *reinterpret_cast<typename Elem<E>::v4*>(p.o + tok * p.o_tok + hq * p.o_head + 4 * c) = out;
}

}  // namespace fa
