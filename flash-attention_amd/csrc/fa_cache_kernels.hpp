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

// Sum over the workgroup of one value per thread, exclusive of the thread's own; `total` for everybody.
template <int THREADS>
__device__ __forceinline__ int64_t exclusive_sum(int64_t v, int64_t* wave_sums, int64_t& total) {
    constexpr int W = THREADS / 64;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t s = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int64_t u = __shfl_up(s, d);
        if (lane >= d) s += u;
    }
    if (lane == 63) wave_sums[wave] = s;
    __syncthreads();
    int64_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        const int64_t x = wave_sums[w];
        if (w < wave) before += x;
        total += x;
    }
    __syncthreads();
    return before + s - v;
}

// The tables of one step.  With h_b keys held, n_b added (or -n_b dropped) and p(x) = ceil(x / page):
//   released_b = max(0, p(h) - p(h + n)),   needed_b = max(0, p(h + n) - p(h));
//   the free list is a stack of c0 pages; all released pages go on it in request order (top = c0 + sum released), then
//   request b takes entries top - 1 - (sum of needed before b) downward.  A request whose pages do not fit (nor
//   its table row, nor its tokens the slot map) is left as it was, and so is every later one that needs pages once the
//   list has run out; q_start counts its tokens all the same, their slots are -1.
// Everything is a running sum over the requests, so every workgroup computes the three sums itself (16 B per
// request, read from the L2) and then fills its share of the outputs: one launch, no
// workgroup waits for another, and no output is an input of another workgroup: a released page that is taken again in
// the same step is found in its old owner's row, not on the stack.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void fa_cache_plan_kernel(const CachePlanParams p) {
    extern __shared__ int lds[];  // token_start[B + 1], need_end[B + 1] and rel_end[B + 1], both with a leading 0
    __shared__ int64_t wave_sums[THREADS / 64];
    __shared__ int taken_s, refused_s;
    int* tok = lds;
    int* need = lds + (p.B + 1);
    int* rel = lds + 2 * (p.B + 1);
    const int tid = threadIdx.x;
    const int per = (p.B + THREADS - 1) / THREADS, b0 = min(tid * per, p.B), b1 = min(b0 + per, p.B);
    const int c0 = clamp_int(p.free_count[0], 0, p.free_cap);
    if (tid == 0) taken_s = refused_s = 0;

    int64_t tokens = 0, released = 0, total_tok, total_rel, total_need;
    for (int b = b0; b < b1; ++b) {
        const int n = p.n_new[b];
        tokens += n > 0 ? n : 0;
        released += plan_row(p.k_len[b], n, p.width, p.log2_page).released();
    }
    tokens = exclusive_sum<THREADS>(tokens, wave_sums, total_tok);
    released = exclusive_sum<THREADS>(released, wave_sums, total_rel);
    auto sat = [](int64_t x) -> int { return x > 0x7fffffffLL ? 0x7fffffff : (int)x; };
    // a request that asks for more than its table row or the slot map holds takes nothing
    auto row_of = [&](int b, int64_t tok_end) -> PlanRow {
        PlanRow r = plan_row(p.k_len[b], p.n_new[b], p.width, p.log2_page);
        if (tok_end > p.max_tokens && p.n_new[b] > 0) r.wide = true;
        if (r.wide) r.after = r.held, r.want = r.have;
        return r;
    };
    int64_t needed = 0, t = tokens;
    for (int b = b0; b < b1; ++b) {
        const int n = p.n_new[b];
        t += n > 0 ? n : 0;
        needed += row_of(b, t).needed();
    }
    needed = exclusive_sum<THREADS>(needed, wave_sums, total_need);
    const int top = c0 + (int)total_rel;
    int taken = 0, refused = 0;
    for (int b = b0; b < b1; ++b) {
        const int n = p.n_new[b];
        tok[b] = sat(tokens);
        tokens += n > 0 ? n : 0;
        const PlanRow r = row_of(b, tokens);
        released += r.released();
        needed += r.needed();
        need[b + 1] = sat(needed);
        rel[b + 1] = sat(released);
        const bool ok = !r.wide && (r.needed() == 0 || needed <= top);
        if (r.needed() > 0 && ok) taken = (int)needed;
        refused += ok ? 0 : 1;
    }
    if (tid == 0) {
        tok[p.B] = sat(total_tok);
        need[0] = rel[0] = 0;
    }
    if (taken) atomicMax(&taken_s, taken);
    if (refused) atomicAdd(&refused_s, refused);
    __syncthreads();
    taken = taken_s;

    const int step = gridDim.x * THREADS, first = blockIdx.x * THREADS + tid;
    // entry i of the pages taken: from the pages released in this step while those last, then from the old stack
    auto page_taken = [&](int i) -> int {
        const int s = top - 1 - i;
        if (s >= c0) {
            const int b = owner_of(rel, p.B, s - c0);
            return p.block_table[b * p.table_stride + row_of(b, tok[b + 1]).want + (s - c0 - rel[b])];
        }
        return s >= 0 ? p.free_pages[s] : -1;
    };
    for (int b = first; b < p.B; b += step) {
        const PlanRow r = row_of(b, tok[b + 1]);
        p.q_start[b] = tok[b];
        const bool ok = !r.wide && (r.needed() == 0 || need[b + 1] <= top);
        p.k_len_out[b] = ok ? r.after : r.held;
    }
    if (first == 0) {
        p.q_start[p.B] = tok[p.B];
        p.counts[0] = min(top - taken, p.free_cap);
        p.counts[1] = refused_s;
    }
    for (int i = first; i < taken; i += step) {
        const int b = owner_of(need, p.B, i);
        p.block_table[b * p.table_stride + row_of(b, tok[b + 1]).have + (i - need[b])] = page_taken(i);
    }
    for (int i = first; i < (int)total_rel && c0 + i < p.free_cap; i += step) {
        const int b = owner_of(rel, p.B, i);
        p.free_pages[c0 + i] = p.block_table[b * p.table_stride + row_of(b, tok[b + 1]).want + (i - rel[b])];
    }
    for (int i = first; i < p.max_tokens; i += step) {
        int slot = -1;
        if (i < tok[p.B]) {
            const int b = owner_of(tok, p.B + 1, i);
            const PlanRow r = row_of(b, tok[b + 1]);
            if (!r.wide && (r.needed() == 0 || need[b + 1] <= top)) {
                const int pos = r.held + (i - tok[b]), j = pos >> p.log2_page;
                const int page = j < r.have ? p.block_table[b * p.table_stride + j] : page_taken(need[b] + j - r.have);
                slot = slot_of(page, pos & ((1 << p.log2_page) - 1), p.log2_page);
            }
        }
        p.slots[i] = slot;
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

// Row t of head h of the new keys (blockIdx.y = 0) or values (1) into its slot, 16 bytes per thread.
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
