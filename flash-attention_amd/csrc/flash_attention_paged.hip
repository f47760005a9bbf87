// Host side of the paged-cache entry points: argument checks, the division of keys over workgroups, launches.  A
// translation unit of its own: it is compiled with NaN honoured (a masked place may hold anything, a visible NaN has to
// come out) and without packed fp32 instructions.
#include "../../include/flash_attention.h"

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <initializer_list>

#include "fa_cache_kernels.hpp"
#include "fa_host.hpp"
#include "fa_shared_prefix_kernel.hpp"

namespace {

using fa_host::fail;

int hip_ok(hipError_t e, const char* what) {
    if (e == hipSuccess) return FA_OK;
    char text[256];
    std::snprintf(text, sizeof(text), "%s failed: %s", what, hipGetErrorString(e));
    return fail(FA_ERR_RUNTIME, text);
}

template <typename F>
int timed(hipStream_t stream, float* elapsed_ms, F&& f) {
    return fa_host::timed(stream, elapsed_ms, [](void* a) -> int { return (*static_cast<F*>(a))(); }, &f);
}

// log2 of a page size that the kernels take, or -1
int log2_page_of(int page_size) {
    for (int l = fa::kMinLog2Page; l <= fa::kMaxLog2Page; ++l)
        if (page_size == 1 << l) return l;
    return -1;
}

bool aligned16(std::initializer_list<const void*> ptrs) {
    for (const void* p : ptrs)
        if (reinterpret_cast<uintptr_t>(p) & 15) return false;
    return true;
}
bool whole_pieces(std::initializer_list<int64_t> strides) {  // 16-byte pieces stay aligned
    for (int64_t s : strides)
        if (s < 0 || s % 8 != 0) return false;
    return true;
}
bool overlap(const void* a, size_t an, const void* b, size_t bn) {
    const auto x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + bn && y < x + an;
}

int check_cache(const fa_paged_cache* c) {
    if (!c || !c->k || !c->v) return fail(FA_ERR_POINTER, "paged cache: null pointer");
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
        return fail(FA_ERR_HEAD_DIM, "paged cache: head_dim must be 64, 128 or 256");
    if (c->heads <= 0 || c->heads > 65535 || c->n_pages <= 0)
        return fail(FA_ERR_SHAPE, "paged cache: n_pages and heads must be positive (at most 65535 heads)");
    if (log2_page_of(c->page_size) < 0)
        return fail(FA_ERR_SHAPE, "paged cache: page_size must be a power of two from 16 to 65536");
    if (!aligned16({c->k, c->v}) ||
        !whole_pieces({c->k_strides[0], c->k_strides[1], c->k_strides[2], c->v_strides[0], c->v_strides[1], c->v_strides[2]}))
        return fail(FA_ERR_SHAPE, "paged cache: k and v must be 16-byte aligned, strides multiples of 8 elements");
    if (c->k_strides[2] < c->head_dim || c->v_strides[2] < c->head_dim)
        return fail(FA_ERR_SHAPE, "paged cache: rows must not overlap");
    if (c->k_strides[2] > (1 << 25) || c->v_strides[2] > (1 << 25))  // (the lanes' offsets within 16 rows are 32-bit)
        return fail(FA_ERR_SHAPE, "paged cache: row strides must be at most 2^25 elements");
    return FA_OK;
}
fa::CacheStrides strides_of(const int64_t (&s)[3]) { return {s[0], s[1], s[2]}; }

constexpr int kMaxKeys = 1 << 30, kMaxBatch = 4000, kMaxGroup = 128;

size_t workspace_of(const fa::LaunchBounds& d, int T, int Hq, int D) {
    return (size_t)T * Hq * ((size_t)d.parts_kept * fa::part_bytes(D) + sizeof(int));
}

int check_shared(int T, int B, int Hq, int Hkv, int prefix_len, int max_k_len) {
    if (T < 0 || B < 0) return fail(FA_ERR_SHAPE, "fa_forward_shared_prefix: T and B must not be negative");
    if (Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0)
        return fail(FA_ERR_SHAPE, "fa_forward_shared_prefix: the query heads must be a multiple of the cache's heads");
    if (Hq / Hkv > kMaxGroup) return fail(FA_ERR_SHAPE, "fa_forward_shared_prefix: at most 128 query heads to a K/V head");
    if (prefix_len < 0 || prefix_len > kMaxKeys || max_k_len < 0 || max_k_len > kMaxKeys)
        return fail(FA_ERR_SEQLEN, "fa_forward_shared_prefix: lengths must be from 0 to 2^30");
    if (B > kMaxBatch) return fail(FA_ERR_SHAPE, "fa_forward_shared_prefix: at most 4000 requests a call");
    if ((int64_t)T * Hq > 0x7fffffffLL / 64 || (int64_t)B * Hq > 0x7fffffffLL / 64)
        return fail(FA_ERR_SHAPE, "fa_forward_shared_prefix: T * Hq or B * Hq too large");
    return FA_OK;
}

template <typename E, int D>
int launch_shared(const fa::SharedPrefixParams& p, const fa::LaunchBounds& d, hipStream_t stream) {
    if (d.blocks > 0x7fffffffLL) return fail(FA_ERR_SHAPE, "fa_forward_shared_prefix: grid size out of range");
    constexpr bool half = std::is_same<E, _Float16>::value;
    void (*const kernel)(fa::SharedPrefixParams) = D == 64    ? (half ? fa::fa_shared_prefix_f16_d64_kernel : fa::fa_shared_prefix_bf16_d64_kernel)
                                                   : D == 128 ? (half ? fa::fa_shared_prefix_f16_d128_kernel : fa::fa_shared_prefix_bf16_d128_kernel)
                                                              : (half ? fa::fa_shared_prefix_f16_d256_kernel : fa::fa_shared_prefix_bf16_d256_kernel);
    hipLaunchKernelGGL(kernel, dim3((unsigned)d.blocks), dim3(256), 0, stream, p);
    if (int rc = hip_ok(hipGetLastError(), "fa_shared_prefix kernel")) return rc;
    constexpr int rows = 256 / (D / 4);
    const int64_t merge = ((int64_t)p.T * p.Hkv * p.g + rows - 1) / rows;
    hipLaunchKernelGGL((fa::fa_shared_prefix_merge_kernel<E, D>), dim3((unsigned)merge), dim3(256), 0, stream, p);
    return hip_ok(hipGetLastError(), "fa_shared_prefix_merge_kernel");
}

}  // namespace

extern "C" {

int fa_cache_plan(const int* k_len, const int* n_new, int* block_table, int64_t table_stride, int* free_pages,
                  const int* free_count, int* q_start, int* k_len_out, int* slots, int* counts, int B, int table_width,
                  int page_size, int free_cap, int max_tokens, void* stream_, float* elapsed_ms) {
    fa_host::clear_error();
    const int log2_page = log2_page_of(page_size);
    if (log2_page < 0) return fail(FA_ERR_SHAPE, "fa_cache_plan: page_size must be a power of two from 16 to 65536");
    if (B <= 0 || B > fa::kMaxPlanRequests) return fail(FA_ERR_SHAPE, "fa_cache_plan: B must be from 1 to 5120");
    if (table_width <= 0 || ((int64_t)table_width << log2_page) > kMaxKeys || (int64_t)B * table_width >= (1 << 30) ||
        table_stride < table_width)
        return fail(FA_ERR_SHAPE, "fa_cache_plan: the block table's rows must be positive, name at most 2^30 keys, and fit their stride");
    if (free_cap < 0 || free_cap > (1 << 30) || max_tokens < 0 || max_tokens > (1 << 30))
        return fail(FA_ERR_SHAPE, "fa_cache_plan: free_cap and max_tokens must be from 0 to 2^30");
    if (!k_len || !n_new || !block_table || !free_count || !q_start || !k_len_out || !counts || (free_cap > 0 && !free_pages) ||
        (max_tokens > 0 && !slots))
        return fail(FA_ERR_POINTER, "fa_cache_plan: null pointer");
    // every workgroup reads all lengths while others write their outputs
    const struct { const void* p; size_t n; } in[] = {{k_len, (size_t)B * 4}, {n_new, (size_t)B * 4}, {free_count, 4}},
        out[] = {{q_start, (size_t)(B + 1) * 4}, {k_len_out, (size_t)B * 4}, {slots, (size_t)max_tokens * 4}, {counts, 8},
                 {free_pages, (size_t)free_cap * 4}, {block_table, ((size_t)(B - 1) * table_stride + table_width) * 4}};
    for (const auto& a : in)
        for (const auto& b : out)
            if (b.n && overlap(a.p, a.n, b.p, b.n))
                return fail(FA_ERR_POINTER, "fa_cache_plan: k_len, n_new and free_count must not overlap what the call writes");
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    fa::CachePlanParams p{k_len, n_new, block_table, table_stride, free_pages, free_count, q_start, k_len_out, slots, counts,
                          B, table_width, log2_page, free_cap, max_tokens};
    // small steps: a smaller workgroup's rounds of sums are quicker; large ones: a thread or two per token and request
    const bool small = B <= 256;
    const int threads = small ? 256 : 1024;
    int64_t blocks = (std::max(max_tokens, B) + threads - 1) / threads;
    if (blocks > 256) blocks = 256;
    return timed(stream, elapsed_ms, [&]() -> int {
        if (small)
            hipLaunchKernelGGL(fa::fa_cache_plan_kernel<256>, dim3((unsigned)blocks), dim3(256), 0, stream, p);
        else
            hipLaunchKernelGGL(fa::fa_cache_plan_kernel<1024>, dim3((unsigned)blocks), dim3(1024), 0, stream, p);
        return hip_ok(hipGetLastError(), "fa_cache_plan_kernel");
    });
}

int fa_cache_write(const uint16_t* dK, const uint16_t* dV, int64_t k_tok, int64_t k_head, int64_t v_tok, int64_t v_head,
                   const fa_paged_cache* cache, const int* slots, int tokens, void* stream_, float* elapsed_ms) {
    fa_host::clear_error();
    if (int rc = check_cache(cache)) return rc;
    if (tokens < 0 || (int64_t)tokens * cache->heads * (cache->head_dim / 8) > 0xffffff00LL)  // (threads of a launch: 32 bits)
        return fail(FA_ERR_SHAPE, "fa_cache_write: tokens must not be negative, tokens * heads * head_dim below 2^35");
    if (elapsed_ms) *elapsed_ms = 0.0f;
    if (tokens == 0) return FA_OK;
    if (!dK || !dV || !slots) return fail(FA_ERR_POINTER, "fa_cache_write: null pointer");
    if (!aligned16({dK, dV}) || !whole_pieces({k_tok, k_head, v_tok, v_head}))
        return fail(FA_ERR_SHAPE, "fa_cache_write: k and v must be 16-byte aligned, strides multiples of 8 elements");
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    const int log2_chunks = cache->head_dim == 64 ? 3 : cache->head_dim == 128 ? 4 : 5;
    fa::CacheWriteParams p{dK, dV, cache->k, cache->v, slots, k_tok, k_head, v_tok, v_head, strides_of(cache->k_strides),
                           strides_of(cache->v_strides), tokens, cache->heads, log2_page_of(cache->page_size), cache->n_pages, log2_chunks};
    const int64_t blocks = (((int64_t)tokens * cache->heads << log2_chunks) + 255) / 256;
    return timed(stream, elapsed_ms, [&]() -> int {
        hipLaunchKernelGGL(fa::fa_cache_write_kernel, dim3((unsigned)blocks, 2), dim3(256), 0, stream, p);
        return hip_ok(hipGetLastError(), "fa_cache_write_kernel");
    });
}

size_t fa_shared_prefix_workspace(int T, int B, int Hq, int Hkv, int D, int prefix_len, int max_k_len) {
    fa_host::clear_error();
    if (T == 0 || B == 0 || (D != 64 && D != 128 && D != 256) || check_shared(T, B, Hq, Hkv, prefix_len, max_k_len) != FA_OK) return 0;
    return workspace_of(fa::launch_bounds_of(T, B, Hkv, Hq / Hkv, D, prefix_len, max_k_len, fa_host::device_cus()), T, Hq, D);
}

int fa_forward_shared_prefix(const uint16_t* dQ, int64_t q_tok, int64_t q_head, uint16_t* dO, int64_t o_tok, int64_t o_head,
                             const fa_paged_cache* cache, const int* prefix_table, int prefix_len, const int* block_table,
                             int64_t table_stride, int table_width, const int* q_start, const int* k_len, int T, int B, int Hq,
                             int dtype, int flags, float scale, int max_k_len, void* workspace, size_t workspace_bytes,
                             void* stream_, float* elapsed_ms) {
    fa_host::clear_error();
    if (int rc = check_cache(cache)) return rc;
    if (dtype != FA_DTYPE_FP16 && dtype != FA_DTYPE_BF16) return fail(FA_ERR_SHAPE, "fa_forward_shared_prefix: unknown dtype");
    if (flags & ~FA_FLAG_CAUSAL) return fail(FA_ERR_SHAPE, "fa_forward_shared_prefix: unknown flag");
    // (a masked score is -inf before it is scaled)
    if (!std::isfinite(scale) || scale < 1e-30f) return fail(FA_ERR_SHAPE, "fa_forward_shared_prefix: scale must be positive and finite");
    const int log2_page = log2_page_of(cache->page_size), Hkv = cache->heads, D = cache->head_dim;
    if (int rc = check_shared(T, B, Hq, Hkv, prefix_len, max_k_len)) return rc;
    if (table_width < 0 || ((int64_t)table_width << log2_page) > kMaxKeys || table_stride < table_width)
        return fail(FA_ERR_SHAPE, "fa_forward_shared_prefix: the block table's rows must name at most 2^30 keys and fit their stride");
    if (elapsed_ms) *elapsed_ms = 0.0f;
    if (T == 0 || B == 0) return FA_OK;
    if (!dQ || !dO || !q_start || !k_len || (prefix_len > 0 && !prefix_table) || (table_width > 0 && !block_table))
        return fail(FA_ERR_POINTER, "fa_forward_shared_prefix: null pointer");
    if (!aligned16({dQ, dO}) || !whole_pieces({q_tok, q_head, o_tok, o_head}))
        return fail(FA_ERR_SHAPE, "fa_forward_shared_prefix: q and o must be 16-byte aligned, strides multiples of 8 elements");
    if (dO == dQ) return fail(FA_ERR_POINTER, "fa_forward_shared_prefix: o must not be q");
    const fa::LaunchBounds d = fa::launch_bounds_of(T, B, Hkv, Hq / Hkv, D, prefix_len, max_k_len, fa_host::device_cus());
    const size_t need = workspace_of(d, T, Hq, D);
    if (need > workspace_bytes || !workspace || !aligned16({workspace})) {
        char text[160];
        std::snprintf(text, sizeof(text), "fa_forward_shared_prefix: the call needs %zu bytes of 16-byte aligned workspace, it got %zu", need,
                      workspace ? workspace_bytes : (size_t)0);
        return fail(FA_ERR_WORKSPACE, text);
    }
    fa::SharedPrefixParams p{};
    p.q = dQ, p.o = dO, p.kc = cache->k, p.vc = cache->v;
    p.q_tok = q_tok, p.q_head = q_head, p.o_tok = o_tok, p.o_head = o_head;
    p.ks = strides_of(cache->k_strides), p.vs = strides_of(cache->v_strides);
    p.prefix_table = prefix_table, p.block_table = block_table, p.table_stride = table_stride;
    p.q_start = q_start, p.k_len = k_len;
    p.part_o = static_cast<float*>(workspace);
    p.part_ml = p.part_o + (size_t)d.parts_kept * T * Hq * D;
    p.row_parts = reinterpret_cast<int*>(p.part_ml + (size_t)d.parts_kept * T * Hq * 2);
    p.T = T, p.B = B, p.Hkv = Hkv, p.g = Hq / Hkv, p.log2_page = log2_page, p.n_pages = cache->n_pages;
    p.prefix_len = prefix_len, p.table_width = table_width, p.causal = flags & FA_FLAG_CAUSAL;
    p.scale_log2e = scale * 1.44269504088896340736f;
    p.rule = d.rule, p.g_reciprocal = fa::group_reciprocal(p.g);
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    return timed(stream, elapsed_ms, [&]() -> int {
        if (dtype == FA_DTYPE_FP16)
            return D == 64 ? launch_shared<_Float16, 64>(p, d, stream) : D == 128 ? launch_shared<_Float16, 128>(p, d, stream)
                                                                                  : launch_shared<_Float16, 256>(p, d, stream);
        return D == 64 ? launch_shared<__bf16, 64>(p, d, stream) : D == 128 ? launch_shared<__bf16, 128>(p, d, stream)
                                                                            : launch_shared<__bf16, 256>(p, d, stream);
    });
}

}  // extern "C"
