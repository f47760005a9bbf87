// Kernels that keep the paged K/V cache: the tables of a serving step from the requests' lengths (fa_cache_plan_kernel)
// and the store of new keys and values through a slot map (fa_cache_write_kernel).  No counterpart in the reference,
// whose tensors are dense [B][H][L][D] (flash_attention_tensor_cores/wrapper.cu:21-34).
#pragma once
#include <hip/hip_runtime.h>

#include "fa_paged_index.hpp"

namespace fa {

typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));

struct CachePlanParams {
    const int* k_len;
    const int* n_new;
    int* block_table;
    int64_t table_stride;
    int* free_pages;
    const int* free_count;
    int* q_start;
    int* k_len_out;
    int* slots;
    int* counts;
    int B, width, log2_page, free_cap, max_tokens;
};

template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_add(int v) { return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, true); }
// Inclusive sum over the wave: within rows of 16 lanes, then row ends into the rows above.
__device__ __forceinline__ int wave_sum_up(int v) {
    v = dpp_add<0x111, 0xf>(v);
    v = dpp_add<0x112, 0xf>(v);
    v = dpp_add<0x114, 0xf>(v);
    v = dpp_add<0x118, 0xf>(v);
    v = dpp_add<0x142, 0xa>(v);
    return dpp_add<0x143, 0xc>(v);
}
// Sums over the workgroup of K values per thread, exclusive of the thread's own; `total` for everybody.  `waves`: K ints a wave.
template <int THREADS, int K>
__device__ __forceinline__ void exclusive_sums(int (&v)[K], int (&total)[K], int* waves) {
    constexpr int W = THREADS / 64;
    static_assert(W <= 16, "the waves' sums are one row of lanes");
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int s = wave_sum_up(v[k]);
        if (lane == 63) waves[k * W + wave] = s;
        v[k] = s - v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int own = lane < W ? waves[k * W + lane] : 0, s = wave_sum_up(own);
        total[k] = __builtin_amdgcn_readlane(s, W - 1);
        v[k] += __builtin_amdgcn_readlane(s - own, __builtin_amdgcn_readfirstlane(wave));
    }
    __syncthreads();
}

// The tables of one step.  With h_b keys held, n_b added (or -n_b dropped) and p(x) = ceil(x / page):
//   released_b = max(0, p(h) - p(h + n)),   needed_b = max(0, p(h + n) - p(h));
//   the free list is a stack of c0 pages; all released pages go on it in request order (top = c0 + sum released), then
//   request b takes entries top - 1 - (sum of needed before b) downward.  A request whose pages do not fit (nor
//   its table row, nor its tokens the slot map) is left as it was, and so is every later one that needs pages once the
//   list has run out; q_start counts its tokens all the same, their slots are -1.
// Everything is a running sum over the requests, so every workgroup computes the sums itself (8 B per request, read from
// the L2) and then fills its share of the outputs: one launch, no workgroup waits for another, and no output is an input
// of another workgroup: a released page that is taken again in the same step is found in its old owner's row, not on the
// stack.  Bound by latency: the lengths' load, two rounds of sums, the search of a token's request in LDS, the load of its
// page.  Measured: 8 requests 2.9 us on the GPU, 1 000 requests 9.1 us a call (LDS scans by doubling steps, lengths read
// twice: 18.7), 4 096 requests 14.2 (28.3).
// (Tokens are summed in two halves of 16 bits: 5120 requests of 2^31 - 1 tokens stay within 31 bits each.)
template <int THREADS>
__global__ __launch_bounds__(THREADS) void fa_cache_plan_kernel(const CachePlanParams p) {
    constexpr int MAXB = THREADS == 256 ? 256 : kMaxPlanRequests, E = (MAXB + THREADS - 1) / THREADS;
    // sums before each request (and their totals): tokens, pages needed, pages released; its keys, -1 - keys where refused
    __shared__ int tok[MAXB + 1], need[MAXB + 1], rel[MAXB + 1], state[MAXB];
    __shared__ int waves[3 * 16], taken_s, refused_s;
    const int tid = threadIdx.x;
    const int per = (p.B + THREADS - 1) / THREADS, b0 = tid * per;
    const int c0 = clamp_int(p.free_count[0], 0, p.free_cap);
    if (tid == 0) taken_s = refused_s = 0;

    int k[E], n[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const bool there = e < per && b0 + e < p.B;
        k[e] = there ? p.k_len[b0 + e] : 0;
        n[e] = there ? p.n_new[b0 + e] : 0;
    }
    int v[3] = {0, 0, 0}, total[3];  // tokens' low and high halves, pages released
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int add = n[e] > 0 ? n[e] : 0;
        v[0] += add & 0xffff;
        v[1] += add >> 16;
        v[2] += plan_row(k[e], n[e], p.width, p.log2_page).released();
    }
    exclusive_sums<THREADS, 3>(v, total, waves);
    auto tokens_of = [](int lo, int hi) -> int64_t { return ((int64_t)hi << 16) + lo; };
    auto sat = [](int64_t x) -> int { return x > 0x7fffffffLL ? 0x7fffffff : (int)x; };
    const int top = c0 + total[2];
    int64_t tokens = tokens_of(v[0], v[1]), end = tokens;
    // a request that asks for more than its table row or the slot map holds takes nothing
    auto row_of = [&](int e, int64_t tok_end) -> PlanRow {
        PlanRow r = plan_row(k[e], n[e], p.width, p.log2_page);
        if (tok_end > p.max_tokens && n[e] > 0) r.wide = true;
        if (r.wide) r.after = r.held, r.want = r.have;
        return r;
    };
    int w[1] = {0}, need_total[1];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        end += n[e] > 0 ? n[e] : 0;
        w[0] += row_of(e, end).needed();
    }
    exclusive_sums<THREADS, 1>(w, need_total, waves);
    int needed = w[0], released = v[2], taken = 0, refused = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int b = b0 + e;
        if (e >= per || b >= p.B) break;
        tok[b] = sat(tokens);
        need[b] = needed;
        rel[b] = released;
        tokens += n[e] > 0 ? n[e] : 0;
        const PlanRow r = row_of(e, tokens);
        released += r.released();
        needed += r.needed();
        const bool ok = !r.wide && (r.needed() == 0 || needed <= top);
        if (r.needed() > 0 && ok) taken = needed;
        refused += ok ? 0 : 1;
        state[b] = ok ? r.held : -1 - r.held;
        if (blockIdx.x == 0) {
            p.q_start[b] = tok[b];
            p.k_len_out[b] = ok ? r.after : r.held;
        }
    }
    if (tid == 0) {
        tok[p.B] = sat(tokens_of(total[0], total[1]));
        need[p.B] = need_total[0];
        rel[p.B] = total[2];
    }
    if (taken) atomicMax(&taken_s, taken);
    if (refused) atomicAdd(&refused_s, refused);
    __syncthreads();
    taken = taken_s;
    if (blockIdx.x == 0 && tid == 0) {
        p.q_start[p.B] = tok[p.B];
        p.counts[0] = min(top - taken, p.free_cap);
        p.counts[1] = refused_s;
    }

    const int step = gridDim.x * THREADS, first = blockIdx.x * THREADS + tid;
    // the pages that request b keeps of those it held before it dropped some
    auto kept = [&](int b) -> int { return plan_row(p.k_len[b], p.n_new[b], p.width, p.log2_page).want; };
    // entry i of the pages taken: from the pages released in this step while those last, then from the old stack
    auto page_taken = [&](int i) -> int {
        const int s = top - 1 - i;
        if (s >= c0) {
            const int b = owner_of(rel, p.B, s - c0);
            return p.block_table[b * p.table_stride + kept(b) + (s - c0 - rel[b])];
        }
        return s >= 0 ? p.free_pages[s] : -1;
    };
    auto held = [&](int b) -> int { return state[b] < 0 ? -1 - state[b] : state[b]; };
    for (int i = first; i < p.max_tokens; i += step) {
        int slot = -1;
        if (i < tok[p.B]) {
            const int b = owner_of(tok, p.B + 1, i);
            if (state[b] >= 0) {
                const int pos = state[b] + (i - tok[b]), j = pos >> p.log2_page, have = pages_for(state[b], p.log2_page);
                const int page = j < have ? p.block_table[b * p.table_stride + j] : page_taken(need[b] + j - have);
                slot = slot_of(page, pos & ((1 << p.log2_page) - 1), p.log2_page);
            }
        }
        p.slots[i] = slot;
    }
    for (int i = first; i < taken; i += step) {
        const int b = owner_of(need, p.B, i);
        p.block_table[b * p.table_stride + pages_for(held(b), p.log2_page) + (i - need[b])] = page_taken(i);
    }
    for (int i = first; i < total[2] && c0 + i < p.free_cap; i += step) {
        const int b = owner_of(rel, p.B, i);
        p.free_pages[c0 + i] = p.block_table[b * p.table_stride + kept(b) + (i - rel[b])];
    }
}

struct CacheWriteParams {
    const uint16_t* k;
    const uint16_t* v;
    uint16_t* kc;
    uint16_t* vc;
    const int* slots;
    int64_t k_tok, k_head, v_tok, v_head;
    CacheStrides ks, vs;
    int tokens, heads, log2_page, n_pages, log2_chunks;  // 2^log2_chunks pieces of 16 bytes per row
};

// Row t of head h of the new keys (blockIdx.y = 0) or values (1) into its slot, 16 bytes per thread: every byte is read
// once and written once, neighbouring lanes share a row, so a row of 128 to 512 bytes is whole cache lines.  Bound by memory: 65 536
// tokens of 8 heads at D = 128 take 86 us, 5.8 TB/s of reads and writes; by the launch below some thousand tokens (3 us).
__global__ __launch_bounds__(256) void fa_cache_write_kernel(const CacheWriteParams p) {
    const bool val = blockIdx.y != 0;
    const uint16_t* src = val ? p.v : p.k;
    uint16_t* dst = val ? p.vc : p.kc;
    const int64_t s_tok = val ? p.v_tok : p.k_tok, s_head = val ? p.v_head : p.k_head;
    const CacheStrides& st = val ? p.vs : p.ks;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, row = i >> p.log2_chunks;
    const int t = (int)(row / p.heads), h = (int)(row - (int64_t)t * p.heads), c = (int)(i & ((1 << p.log2_chunks) - 1));
    if (t >= p.tokens) return;
    const int slot = p.slots[t];
    if (slot < 0 || !page_ok(slot >> p.log2_page, p.n_pages)) return;
    const u32x4_t x = *reinterpret_cast<const u32x4_t*>(src + t * s_tok + h * s_head + c * 8);
    *reinterpret_cast<u32x4_t*>(dst + cache_offset(st, slot >> p.log2_page, h, slot & ((1 << p.log2_page) - 1)) + c * 8) = x;
}

}  // namespace fa
