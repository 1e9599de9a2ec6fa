// The paged key-value cache as its kernels see it, and the host checks that every entry point makes of a kx_kv.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

#include "kx_kernels.h"

namespace kx {

constexpr int KV_MAX_PAGE = 1024;

inline int kv_elem_bytes(int type) { return type == KX_KV_F32 ? 4 : 2; }

// the description can be used: sizes, alignment, pages and layers that do not overlap
inline bool kv_ok(const kx_kv* c) {
    if (!c || c->type < KX_KV_F32 || c->type > KX_KV_BF16) return false;
    if (c->layers < 1 || c->n_pages < 1 || c->heads < 1 || c->dk < 1 || c->dv < 1 || c->n_seqs < 1 || c->max_pages < 1) return false;
    if (c->page < 1 || c->page > KV_MAX_PAGE || (c->page & (c->page - 1)) || c->dk > 1024 || c->dv > 1024) return false;
    if (c->heads > 1 << 16 || c->n_pages > 1 << 30 || static_cast<long>(c->max_pages) * c->page > INT32_MAX) return false;
    // slots and table entries are walked in 32 bits, up to a CTA's width at a time
    if (c->n_seqs > 1 << 30 || c->max_pages > INT32_MAX - 1024) return false;
    if (!c->k || !c->v || !c->table || !c->lens || !c->refs) return false;
    const long sz = kv_elem_bytes(c->type);
    if (c->dk * sz % 16 || c->dv * sz % 16) return false;
    if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15) return false;
    const long kpage = static_cast<long>(c->heads) * c->page * c->dk, vpage = static_cast<long>(c->heads) * c->page * c->dv;
    if (kpage > (1l << 28) || vpage > (1l << 28)) return false;  // a page's bytes are counted in 32 bits
    const auto strides_ok = [&](long st_page, long st_layer, long need) {
        // extents of up to 2^60 elements: no product below, or in a kernel, passes 64 bits
        if (st_page < need || st_page > (1l << 60) / c->n_pages || st_page * sz % 16) return false;
        if (c->layers == 1) return true;
        if (st_layer < need || st_layer > (1l << 60) / c->layers || st_layer * sz % 16) return false;
        // either each layer is a pool of its own or each page holds its layers one after another
        return st_layer >= (c->n_pages - 1) * st_page + need || st_page >= (c->layers - 1) * st_layer + need;
    };
    return strides_ok(c->k_page, c->k_layer, kpage) && strides_ok(c->v_page, c->v_layer, vpage);
}

__device__ __forceinline__ void kv_report(int* status, int bit) {
    if (status) atomicOr(status, bit);
}

}  // namespace kx
