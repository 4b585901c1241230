// Shared by the kernels of the paged cache (cache.cu, draft_attn.cu): positions to pages, argument checks.
#pragma once
#include "common.cuh"

namespace htree {

// n / d for 0 <= n < 2^31 by one multiplication: with 2^(s-1) < d <= 2^s and m = ceil(2^(31+s) / d) the error n*(m*d - 2^(31+s)) / d
// stays below 2^(31+s), a whole unit of the quotient being d times that.
struct FastDiv {
    uint32_t mul, shift, d;
    FastDiv() = default;
    explicit FastDiv(uint32_t d_) : d(d_) {
        uint32_t s = 0;
        while ((uint64_t(1) << s) < d_) ++s;
        mul = (uint32_t)(((uint64_t(1) << (31 + s)) + d_ - 1) / d_);
        shift = 31 + s;
    }
    __device__ __forceinline__ uint32_t div(uint32_t n) const { return (uint32_t)(((uint64_t)n * mul) >> shift); }
};

inline int cache_esize(int dtype) { return dtype == HTREE_F32 ? 4 : 2; }
inline bool cache_aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
// strides (elements) of three leading dimensions whose rows have to start on 16 bytes
inline bool cache_strides_ok(const int64_t* s, int es) {
    for (int i = 0; i < 3; ++i) if (s[i] < 0 || (s[i] * es) % 16 != 0) return false;
    return true;
}
inline int check_cache(const HtreeCache* c) {
    if (!c || !c->k || !c->v) return HTREE_E_NULL;
    if (c->dtype != HTREE_F32 && c->dtype != HTREE_BF16 && c->dtype != HTREE_F16) return HTREE_E_DTYPE;
    if (c->pages <= 0 || c->page_size <= 0 || c->H_kv <= 0 || c->K <= 0 || c->V <= 0) return HTREE_E_SHAPE;
    if (c->K % 8 || c->V % 8 || !cache_aligned(c->k) || !cache_aligned(c->v)) return HTREE_E_ALIGN;
    const int64_t ks[3] = {c->k_page, c->k_row, c->k_head}, vs[3] = {c->v_page, c->v_row, c->v_head};
    const int es = cache_esize(c->dtype);
    if (!cache_strides_ok(ks, es) || !cache_strides_ok(vs, es)) return HTREE_E_ALIGN;
    return 0;
}

int sm_count();      // of the current device (cache.cu)

}  // namespace htree
