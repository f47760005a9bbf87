// Attention of a batch whose requests share a long prefix, over a paged K/V cache.  Row (t, h), token t of request b and
// query head h of K/V head h / g:
//     O = sum_j p_j V_j / sum_j p_j,   p_j = exp(scale Q.K_j),   j over the Lp keys of the prefix and over the request's
//     own keys j <= k_len[b] - n[b] + (t - q_start[b])  (causal; all k_len[b] of them otherwise).
// The sum over j falls into parts that are computed apart and joined by their maxima (log-sum-exp): the prefix part is one
// matrix product for the whole batch, its rows being the g heads of ALL tokens stacked up against each K/V head, so the
// prefix is read from memory once per 128 stacked rows instead of once per request; the own part has the rows of one
// request.  Both parts are divided over ranges of keys until the chip is full.
// A workgroup has 4 waves of 32 rows and walks its range in tiles of kTk keys (transposed scores S^T = K.Q^T, the score
// registers rounded to 16 bits as B operand of O^T += V^T.P^T, swizzled LDS tiles: the lane geometry of
// fa_fwd_general_kernel.hpp).  fa_shared_prefix_merge_kernel joins the parts.
//
// Masks.  A tile that holds a masked place for some row of the wave (the end of the range, the causal diagonal, a page that
// is none) takes the masked form of the step: scores of masked places become -inf whatever K holds there, and V is
// multiplied with its infinities and NaN taken out (0 x NaN is NaN), which are then added to the rows that do see them.
// Rows that see no key give 0.
#pragma once
#include "fa_fwd_general_kernel.hpp"
#include "fa_fwd_ring_kernel.hpp"  // wait_all_vmem
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
    int slots;                      // workgroups that the chip holds at a time
    int max_prefix_parts, max_own_parts;
};

template <typename E>
struct Elem;
template <>
struct Elem<_Float16> {
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    typedef _Float16 v4 __attribute__((ext_vector_type(4)));
    static constexpr unsigned kExpMask = 0x7c00;
    static __device__ __forceinline__ f32x16 mfma(v8 a, v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <>
struct Elem<__bf16> {
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    typedef __bf16 v4 __attribute__((ext_vector_type(4)));
    static constexpr unsigned kExpMask = 0x7f80;
    static __device__ __forceinline__ f32x16 mfma(v8 a, v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};

// max that keeps NaN (v_maximum3_f32): a row that sees a NaN score is NaN, and no operand is canonicalised first.
__device__ __forceinline__ float max_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// Infinities and NaN of a V fragment: taken out (returned fragment), and their places (kind 1 NaN, 2 +inf, 3 -inf) as ones.
template <typename E>
__device__ __forceinline__ typename Elem<E>::v8 finite_part(typename Elem<E>::v8 x, bool& special) {
    u32x4 u = __builtin_bit_cast(u32x4, x);
    constexpr unsigned m = Elem<E>::kExpMask;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if ((u[i] & m) == m) u[i] &= 0xffff0000u, special = true;
        if ((u[i] & (m << 16)) == m << 16) u[i] &= 0x0000ffffu, special = true;
    }
    return __builtin_bit_cast(typename Elem<E>::v8, u);
}
template <typename E>
__device__ __forceinline__ typename Elem<E>::v8 special_part(typename Elem<E>::v8 x, int kind) {
    const u32x4 u = __builtin_bit_cast(u32x4, x);
    constexpr unsigned m = Elem<E>::kExpMask;
    typename Elem<E>::v8 r;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const unsigned h = (u[i / 2] >> (16 * (i & 1))) & 0xffffu, a = h & 0x7fffu;
        const int k = a > m ? 1 : a < m ? 0 : h == a ? 2 : 3;
        r[i] = (E)(k == kind ? 1.0f : 0.0f);
    }
    return r;
}

template <int D>
struct SharedCfg;
template <>
struct SharedCfg<64> {
    static constexpr int kTk = 64, kStages = 4, kOcc = 2;  // 16 KiB a stage
};
template <>
struct SharedCfg<128> {
    static constexpr int kTk = 32, kStages = 4, kOcc = 2;  // 16 KiB
};
template <>
struct SharedCfg<256> {
    static constexpr int kTk = 32, kStages = 4, kOcc = 1;  // 32 KiB
};

// The division of a launch into workgroups, from the requests' lengths; every workgroup computes it for itself.
//   A request with fewer than 128 rows (new tokens x g) is short: its rows are stacked up with those of the other short
// requests against the prefix (items of kind P: one K/V head, 128 stacked rows, a range of the prefix) and alone against
// its own keys (O: one head, the request's rows, a range of its keys).  A longer request fills row tiles of its own, which walk
// prefix and own keys in one go (J: one head, 128 of its rows, a range of both): nothing is gained by stacking.
//   Ranges are `steps` key tiles long, up to half a range more or less: all tiles of the launch over the workgroups that
// the chip holds.
struct SharedPlan {
    int stacked;        // rows of the short requests, per K/V head
    int prefix_tiles;   // key tiles of the prefix
    int prefix_parts;   // ranges of the prefix that P items walk
    int p_items;
    int steps;
};

// Inclusive sum over the 256 threads of a workgroup; `total` for everybody.  `tmp`: 4 ints of LDS.
__device__ __forceinline__ int workgroup_sum(int v, int* tmp, int& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int u = __shfl_up(v, d);
        if (lane >= d) v += u;
    }
    __syncthreads();
    if (lane == 63) tmp[wave] = v;
    __syncthreads();
    const int a = tmp[0], b = tmp[1], c = tmp[2];
    total = a + b + c + tmp[3];
    return v + (wave > 0 ? a : 0) + (wave > 1 ? b : 0) + (wave > 2 ? c : 0);
}

struct SharedRequest {
    int tok0, n, keys;
};
__device__ __forceinline__ SharedRequest shared_request(const SharedPrefixParams& p, int b) {
    SharedRequest r;
    r.tok0 = clamp_int(p.q_start[b], 0, p.T);
    r.n = clamp_int(p.q_start[b + 1], r.tok0, p.T) - r.tok0;
    r.keys = clamp_int(p.k_len[b], 0, p.table_width << p.log2_page);
    return r;
}

// Items of a request; 0 where it has no rows.
template <int TK>
__device__ __forceinline__ int request_items(const SharedPrefixParams& p, const SharedPlan& s, const SharedRequest& r, int& tiles, int& parts) {
    const int rows = r.n * p.g, own = (r.keys + TK - 1) / TK;
    tiles = (rows + 127) >> 7;
    parts = rows >= 128 ? parts_for(s.prefix_tiles + own, s.steps, p.max_prefix_parts + p.max_own_parts) : parts_for(own, s.steps, p.max_own_parts);
    return tiles * parts * p.Hkv;
}

// LDS: stacked_start[B] (stacked tokens before request b), item_start[B] (items before it, P items among them).
template <int TK>
__device__ __forceinline__ int shared_plan(const SharedPrefixParams& p, SharedPlan& s, int* stacked_start, int* item_start, int* tmp) {
    s.prefix_tiles = (p.prefix_len + TK - 1) / TK;
    int tokens = 0;
    float work = 0.0f;  // key tiles of all row tiles, per K/V head
    for (int b0 = 0; b0 < p.B; b0 += 256) {
        const int b = b0 + (int)threadIdx.x;
        int n = 0;
        if (b < p.B) {
            const SharedRequest r = shared_request(p, b);
            const int rows = r.n * p.g, own = (r.keys + TK - 1) / TK;
            if (rows < 128) n = r.n;
            work += (float)((rows + 127) >> 7) * (float)(own + (rows < 128 ? 0 : s.prefix_tiles));
        }
        int total;
        const int sum = workgroup_sum(n, tmp, total);
        if (b < p.B) stacked_start[b] = tokens + sum - n;
        tokens += total;
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) work += __shfl_xor(work, d);
    float* ftmp = reinterpret_cast<float*>(tmp);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) ftmp[threadIdx.x >> 6] = work;
    __syncthreads();
    work = ftmp[0] + ftmp[1] + ftmp[2] + ftmp[3];
    s.stacked = tokens * p.g;
    const int p_tiles = (s.stacked + 127) >> 7;
    work += (float)p_tiles * (float)s.prefix_tiles;
    s.steps = steps_for(work, p.Hkv, p.slots, 128 / TK);
    s.prefix_parts = s.prefix_tiles > 0 && p_tiles > 0 ? parts_for(s.prefix_tiles, s.steps, p.max_prefix_parts) : 0;
    s.p_items = p_tiles * s.prefix_parts * p.Hkv;
    int items = s.p_items;
    for (int b0 = 0; b0 < p.B; b0 += 256) {
        const int b = b0 + (int)threadIdx.x;
        int n = 0, tiles, parts;
        if (b < p.B) n = request_items<TK>(p, s, shared_request(p, b), tiles, parts);
        int total;
        const int sum = workgroup_sum(n, tmp, total);
        if (b < p.B) item_start[b] = items + sum - n;
        items += total;
    }
    __syncthreads();
    return items;
}

// Item x of units x tiles: eight units at a time, tile by tile, so that the row tiles that read the same keys (one unit: a
// K/V head and a range) follow each other on one XCD (workgroup ids congruent mod 8 share one and its L2).
__device__ __forceinline__ void unit_and_tile(int x, int units, int tiles, int& unit, int& tile) {
    const int full = units >> 3, per = 8 * tiles;
    const int grp = min(x / per, full), r = x - grp * per, w = grp < full ? 8 : units & 7;
    tile = r / w;
    unit = grp * 8 + (r - tile * w);
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

template <typename E, int D>
__global__ __launch_bounds__(256, SharedCfg<D>::kOcc) void fa_shared_prefix_kernel(const SharedPrefixParams p) {
    using HD = HeadDim<D>;
    using CFG = SharedCfg<D>;
    using v8 = typename Elem<E>::v8;
    constexpr int TK = CFG::kTk, KB = TK / 32, ST = CFG::kStages, kTile = TK * HD::kRow, kStage = 2 * kTile;
    constexpr int PPW = kTile / 1024 / 4;            // 1 KiB pieces of a K (or V) tile that each wave moves
    constexpr int RPP = 1024 / HD::kRow;             // rows per piece
    constexpr int RPW = RPP * PPW;                   // rows per wave and tile: 16 (D = 64) or 8, on one page
    constexpr int CPT = TK / 16;                     // 16-key groups per tile
    __shared__ __attribute__((aligned(1024))) char ring[ST * kStage];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const LaneGeomD<D> geo = make_lane_geom_d<D>(lane);
    const int P1 = (1 << p.log2_page) - 1;  // (row in a page)

    // ---- which rows against which keys: rows row0 .. of a request's `rows` (or of the stacked ones) against key tiles
    //      u0 .. of the sequence of the prefix' tiles and the request's own
    SharedPlan plan;
    int head, part, parts, row0, rows, u0, n_tiles, own_keys = 0, n_tok = 0, tok;
    bool stacked;
    const int* own_table = nullptr;
    const int R_off = wave * 32 + geo.r;
    {
        int* stacked_start = reinterpret_cast<int*>(ring);  // (free until the first transfer)
        int* item_start = stacked_start + p.B;
        __shared__ int tmp[4];
        const int x = (int)blockIdx.x;
        if (x >= shared_plan<TK>(p, plan, stacked_start, item_start, tmp)) return;
        int unit, tile, u1;
        stacked = x < plan.p_items;
        if (stacked) {
            parts = plan.prefix_parts;
            unit_and_tile(x, p.Hkv * parts, (plan.stacked + 127) >> 7, unit, tile);
            head = unit / parts, part = unit - head * parts;
            row0 = tile * 128, rows = plan.stacked;
            u0 = (int)((int64_t)plan.prefix_tiles * part / parts);
            u1 = (int)((int64_t)plan.prefix_tiles * (part + 1) / parts);
            const int t = min(row0 + R_off, rows - 1) / p.g;  // stacked token
            const int b = owner_of(stacked_start, p.B, t);
            tok = clamp_int(p.q_start[b], 0, p.T) + t - stacked_start[b];
        } else {
            const int b = last_at_most(item_start, p.B, x);
            const SharedRequest r = shared_request(p, b);
            int tiles;
            request_items<TK>(p, plan, r, tiles, parts);
            unit_and_tile(x - item_start[b], p.Hkv * parts, tiles, unit, tile);
            head = unit / parts, part = unit - head * parts;
            row0 = tile * 128, rows = r.n * p.g, n_tok = r.n;
            own_keys = r.keys;
            own_table = p.block_table + b * p.table_stride;
            tok = r.tok0 + min(row0 + R_off, rows - 1) / p.g;
            // no row of the tile sees further than its last one
            const int last_ti = (min(row0 + 128, rows) - 1) / p.g, see = p.causal ? min(r.keys, r.keys - r.n + last_ti + 1) : r.keys;
            const int first = rows >= 128 ? 0 : plan.prefix_tiles, n = plan.prefix_tiles + (max(see, 0) + TK - 1) / TK - first;
            u0 = first + (int)((int64_t)n * part / parts);
            u1 = first + (int)((int64_t)n * (part + 1) / parts);
        }
        n_tiles = u1 - u0;
        __syncthreads();  // (the tables above have been read)
    }
    const bool valid = row0 + R_off < rows, wave_valid = row0 + wave * 32 < rows;
    const int R = min(row0 + R_off, rows - 1), ti = R / p.g, hq = head * p.g + (R - ti * p.g), Hq = p.Hkv * p.g;
    const int own_limit = p.causal ? min(own_keys - 1, own_keys - n_tok + ti) : own_keys - 1;  // the last own key this row sees

    // ---- transfers: this wave moves rows RPW * wave .. of each tile.  They lie on one page, whose number is uniform: lane L
    //      holds the entry of the 16-key group group0 + L of the range, 64 groups at a time (the next 64 are loaded one
    //      refill ahead).  Lane l fills slot l % kChunks of row l / kChunks of a piece with the chunk the swizzle maps there.
    const unsigned ring_lds = __builtin_amdgcn_readfirstlane((unsigned)(size_t)(__attribute__((address_space(3))) char*)ring);
    const int d_rip = lane / HD::kChunks, d_slot = lane % HD::kChunks;
    unsigned k_off[PPW], v_off[PPW];
#pragma unroll
    for (int j = 0; j < PPW; ++j) {
        const int row = RPW * wave + RPP * j + d_rip;
        k_off[j] = (unsigned)((RPP * j + d_rip) * (int)p.ks.row * 2) + (unsigned)((d_slot ^ (row & HD::kKMask)) << 4);
        v_off[j] = (unsigned)((RPP * j + d_rip) * (int)p.vs.row * 2) + (unsigned)((d_slot ^ ((row & HD::kVMask) << 2)) << 4);
    }
    const char* k_head = reinterpret_cast<const char*>(p.kc + head * p.ks.head);
    const char* v_head = reinterpret_cast<const char*>(p.vc + head * p.vs.head);
    const int own_entries = p.table_width, prefix_entries = pages_for(p.prefix_len, p.log2_page);
    auto load_pages = [&](int group) -> int {  // -1: no page
        const int i = group + lane, u = u0 + i / CPT, key = (u < plan.prefix_tiles ? u : u - plan.prefix_tiles) * TK + 16 * (i % CPT);
        const int* table = u < plan.prefix_tiles ? p.prefix_table : own_table;
        const int j = key >> p.log2_page;
        const int page = i < n_tiles * CPT && j < (u < plan.prefix_tiles ? prefix_entries : own_entries) ? table[j] : -1;
        return page_ok(page, p.n_pages) ? page : -1;
    };
    int pages = 0, pages_next = 0;
    unsigned on_page = 0;  // CPT bits per tile sent for and not yet computed: the groups that lie on a page
    auto send = [&](int t) {
        const int g0 = t * CPT;
        if ((g0 & 63) == 0) {
            pages = t == 0 ? load_pages(0) : pages_next;
            pages_next = g0 + 64 < n_tiles * CPT ? load_pages(g0 + 64) : -1;
        }
        on_page |= ((unsigned)(__ballot(pages >= 0) >> (g0 & 63)) & ((1u << CPT) - 1)) << (CPT * (ST - 1));
        // (a group on no page is fetched from page 0: its scores are masked)
        const int page = max(__builtin_amdgcn_readlane(pages, (g0 + wave * RPW / 16) & 63), 0);
        const int u = u0 + t, row = ((u < plan.prefix_tiles ? u : u - plan.prefix_tiles) * TK + wave * RPW) & P1;
        const char* kb = k_head + 2 * ((int64_t)page * p.ks.page + (int64_t)row * p.ks.row);
        const char* vb = v_head + 2 * ((int64_t)page * p.vs.page + (int64_t)row * p.vs.row);
        const unsigned l = ring_lds + (unsigned)(t % ST) * kStage + (unsigned)(PPW * wave) * 1024u;
#pragma unroll
        for (int j = 0; j < PPW; ++j) dma16(l + 1024u * j, kb, k_off[j]);
#pragma unroll
        for (int j = 0; j < PPW; ++j) dma16(l + kTile + 1024u * j, vb, v_off[j]);
    };

#pragma unroll
    for (int t = 0; t < ST - 1; ++t) {
        if (t < n_tiles) send(t);
        on_page >>= CPT;
    }

    v8 qf[HD::kSteps];
    {
        const uint16_t* qr = p.q + tok * p.q_tok + hq * p.q_head + geo.hh * 8;
#pragma unroll
        for (int ks = 0; ks < HD::kSteps; ++ks) qf[ks] = *reinterpret_cast<const v8*>(qr + ks * 16);
    }

    f32x16 oacc[HD::kBlocks];
    float m_run = -1e30f, l_run = 0.0f;
#pragma unroll
    for (int db = 0; db < HD::kBlocks; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e) oacc[db][e] = 0.0f;

    auto v_frag = [&](const char* vb, int kk, int db) -> v8 {
        const char* a0 = vb + geo.v_rd[db] + kk * 16 * HD::kRow;
        const short4_t t0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t*)(a0));
        const short4_t t1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t*)(a0 + 8 * HD::kRow));
        return __builtin_bit_cast(v8, __builtin_shufflevector(t0, t1, 0, 1, 2, 3, 4, 5, 6, 7));
    };

    wait_all_vmem();
    __syncthreads();
    for (int t = 0; t < n_tiles; ++t) {
        const unsigned groups = on_page & ((1u << CPT) - 1);
        if (t + ST - 1 < n_tiles) send(t + ST - 1);  // into the stage of tile t - 1, which every wave has left
        on_page >>= CPT;
        const int u = u0 + t;
        // the last key of this tile that the row sees; a wave whose rows see none of it passes it by
        const int lim = u < plan.prefix_tiles ? p.prefix_len - 1 - u * TK : own_limit - (u - plan.prefix_tiles) * TK;
        if (wave_valid && __any(lim >= 0)) {
            const char* kb = ring + (t % ST) * kStage;
            const char* vb = kb + kTile;
            f32x16 s[KB];
#pragma unroll
            for (int b = 0; b < KB; ++b) {
#pragma unroll
                for (int e = 0; e < 16; ++e) s[b][e] = 0.0f;
#pragma unroll
                for (int ks = 0; ks < HD::kSteps; ++ks)
                    s[b] = Elem<E>::mfma(*reinterpret_cast<const v8*>(kb + geo.k_rd[ks] + b * 32 * HD::kRow), qf[ks], s[b]);
            }
            const bool masked = __any(lim < TK - 1) || groups != (1u << CPT) - 1;
            if (masked) {
#pragma unroll
                for (int b = 0; b < KB; ++b)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const int k = 32 * b + 8 * (e >> 2) + (e & 3);
                        if (k + 4 * geo.hh > lim || !((groups >> (k >> 4)) & 1)) s[b][e] = -__builtin_inff();
                    }
            }
            float mx = s[0][0];
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
                for (int e = b == 0 ? 1 : 0; e < 16; ++e) mx = max_nan(mx, s[b][e]);
            {
                float a, b;
                half_wave_pair(mx, a, b);
                mx = max_nan(a, b) * p.scale_log2e;
            }
            if (!__all(mx - m_run <= kRescaleSlack)) {
                const float m_new = max_nan(m_run, mx), alpha = __builtin_amdgcn_exp2f(m_run - m_new);
                m_run = m_new;
                l_run *= alpha;
#pragma unroll
                for (int db = 0; db < HD::kBlocks; ++db)
#pragma unroll
                    for (int e = 0; e < 16; ++e) oacc[db][e] *= alpha;
            }
            v8 pf[2 * KB];
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][e], p.scale_log2e, -m_run));
                    l_run += x;
                    pf[2 * b + e / 8][e % 8] = (E)x;
                }
            if (!masked) {
#pragma unroll
                for (int kk = 0; kk < 2 * KB; ++kk)
#pragma unroll
                    for (int db = 0; db < HD::kBlocks; ++db) oacc[db] = Elem<E>::mfma(v_frag(vb, kk, db), pf[kk], oacc[db]);
            } else {
                bool special = false;
#pragma unroll
                for (int kk = 0; kk < 2 * KB; ++kk)
#pragma unroll
                    for (int db = 0; db < HD::kBlocks; ++db)
                        oacc[db] = Elem<E>::mfma(finite_part<E>(v_frag(vb, kk, db), special), pf[kk], oacc[db]);
                if (__any(special)) {
                    v8 sees[2 * KB];  // 1 where the row sees the key
#pragma unroll
                    for (int kk = 0; kk < 2 * KB; ++kk)
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const int k = 16 * kk + 8 * (i >> 2) + (i & 3);
                            sees[kk][i] = (E)(k + 4 * geo.hh <= lim && ((groups >> (k >> 4)) & 1) ? 1.0f : 0.0f);
                        }
#pragma unroll 1
                    for (int kind = 1; kind <= 3; ++kind) {
                        const unsigned bits = kind == 1 ? 0x7fc00000u : kind == 2 ? 0x7f800000u : 0xff800000u;
#pragma unroll
                        for (int db = 0; db < HD::kBlocks; ++db) {
                            f32x16 n;
#pragma unroll
                            for (int e = 0; e < 16; ++e) n[e] = 0.0f;
#pragma unroll
                            for (int kk = 0; kk < 2 * KB; ++kk)
                                n = Elem<E>::mfma(special_part<E>(v_frag(vb, kk, db), kind), sees[kk], n);
#pragma unroll
                            for (int e = 0; e < 16; ++e)
                                if (n[e] > 0.0f) oacc[db][e] += __builtin_bit_cast(float, bits);
                        }
                    }
                }
            }
        }
        // this wave's share of tile t + 1 has landed (transfers complete in order); the next ST - 2 stay in flight
        if (t + ST - 1 < n_tiles)
            asm volatile("s_waitcnt vmcnt(%0)" : : "n"((ST - 2) * 2 * PPW) : "memory");
        else
            wait_all_vmem();
        __syncthreads();
    }

    if (!valid) return;
    const int64_t all = (int64_t)p.T * Hq, row = (int64_t)tok * Hq + hq;
    float l0, l1;
    half_wave_pair(l_run, l0, l1);
    const float l = l0 + l1;
    // (a short request's rows have the P items' parts in front of their own)
    const int before = stacked || rows >= 128 ? 0 : plan.prefix_parts;
    if (!stacked && part == 0 && geo.hh == 0) p.row_parts[row] = before + parts == 1 ? 0 : before + parts;
    if (!stacked && before + parts == 1) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        uint16_t* og = p.o + tok * p.o_tok + hq * p.o_head;
#pragma unroll
        for (int db = 0; db < HD::kBlocks; ++db)
#pragma unroll
            for (int g4 = 0; g4 < 4; ++g4) {
                typename Elem<E>::v4 x;
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = (E)(oacc[db][4 * g4 + e] * inv);
                *reinterpret_cast<typename Elem<E>::v4*>(og + 32 * db + 8 * g4 + 4 * geo.hh) = x;
            }
        return;
    }
    const int64_t slot = (before + part) * all + row;
    if (geo.hh == 0) *reinterpret_cast<f32x2*>(p.part_ml + 2 * slot) = f32x2{m_run, l};
    if (n_tiles == 0) return;  // (nothing is read of a part whose sum is 0)
    float* oa = p.part_o + slot * D;
#pragma unroll
    for (int db = 0; db < HD::kBlocks; ++db)
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4) {
            const f32x4 x = {oacc[db][4 * g4], oacc[db][4 * g4 + 1], oacc[db][4 * g4 + 2], oacc[db][4 * g4 + 3]};
            *reinterpret_cast<f32x4*>(oa + 32 * db + 8 * g4 + 4 * geo.hh) = x;
        }
}

// O = sum_s w_s o_s / sum_s w_s l_s,  w_s = exp2(m_s - max_s m_s): D / 4 lanes per row, four parts in flight.  Rows of no
// request and rows that are written already are left alone.
template <typename E, int D>
__global__ __launch_bounds__(256) void fa_shared_prefix_merge_kernel(const SharedPrefixParams p) {
    constexpr int LPR = D / 4, RPB = 256 / LPR, U = 4;
    const int c = threadIdx.x % LPR, Hq = p.Hkv * p.g;
    const int64_t rows = (int64_t)p.T * Hq, i = (int64_t)blockIdx.x * RPB + threadIdx.x / LPR;
    if (i >= rows) return;
    const int tok = (int)(i / Hq), hq = (int)(i - (int64_t)tok * Hq);
    const int first = p.q_start[0], last = p.q_start[p.B], parts = min(p.row_parts[i], p.max_prefix_parts + p.max_own_parts);
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
