// KERNIX-B200 pages of a key-value cache: room for new tokens (extend), their rows (append), shared copies of sequences
// (fork), release (free) and moving the live pages together (compact). include/kx_kernels.h states what each does.
//
// All of it is bookkeeping on a few hundred KB of integers (latency) plus copies of whole pages or rows (HBM). What has
// to be decided in order -- which free page goes to whom -- is decided by one CTA, whose warps each hold 1024
// reference counts in registers: a count per warp, one scan over the 32 counts, then every page's rank by shuffles.
// What can be done in any order (copying pages, filling table rows) is left to a second launch over the whole GPU,
// which finds the first one's decisions in the workspace (programmatic dependent launch: its CTAs are up by then).
// Integer atomics only where their order cannot show: counts of references, and minima.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdint>

#include "kx_kernels.h"
#include "kx_kv.cuh"
#include "kx_pdl.cuh"

namespace {

constexpr int PLAN = 1024;  // threads of the one-CTA planners
constexpr unsigned FULL = 0xFFFFFFFFu;

// inclusive sum over the CTA's PLAN threads; tmp: 32 words of shared memory. *total: the sum over all.
__device__ __forceinline__ long long block_scan(long long v, long long* tmp, long long* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const long long u = __shfl_up_sync(FULL, v, d);
        if (lane >= d) v += u;
    }
    __syncthreads();  // the readers of an earlier scan are done with tmp
    if (lane == 31) tmp[warp] = v;
    __syncthreads();
    if (warp == 0) {
        long long t = tmp[lane];
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const long long u = __shfl_up_sync(FULL, t, d);
            if (lane >= d) t += u;
        }
        tmp[lane] = t;
    }
    __syncthreads();
    *total = tmp[31];
    return v + (warp ? tmp[warp - 1] : 0);
}

// 1024 pages per warp in registers, so that a pass over up to 32768 pages waits for memory once
constexpr int SEG = 1024, ROUND = 32 * SEG;
struct Seg {
    int4 r[8];  // pages first + 128 u + 4 lane ..
    long first;
};
__device__ __forceinline__ int zeros(int4 r) { return (r.x == 0) + (r.y == 0) + (r.z == 0) + (r.w == 0); }
__device__ __forceinline__ int load_seg(const int32_t* refs, int n, long first, Seg* s) {  // returns the warp's free pages
    const int lane = threadIdx.x & 31;
    const bool vec = (reinterpret_cast<uintptr_t>(refs) & 15) == 0;
    s->first = first;
#pragma unroll
    for (int u = 0; u < 8; u++) {
        const long p = first + u * 128 + lane * 4;
        int4 r = make_int4(1, 1, 1, 1);  // behind the last page: not free
        if (vec && p + 3 < n) {
            r = __ldcg(reinterpret_cast<const int4*>(refs + p));
        } else {
            if (p < n) r.x = __ldcg(refs + p);
            if (p + 1 < n) r.y = __ldcg(refs + p + 1);
            if (p + 2 < n) r.z = __ldcg(refs + p + 2);
            if (p + 3 < n) r.w = __ldcg(refs + p + 3);
        }
        s->r[u] = r;
    }
    int c = 0;
#pragma unroll
    for (int u = 0; u < 8; u++) c += zeros(s->r[u]);
    return __reduce_add_sync(FULL, c);
}

// the number of free pages; every thread of the CTA takes part, tmp: 32 words of shared memory
__device__ __forceinline__ int count_free(const int32_t* refs, int n, int* tmp) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Seg s;
    int mine = 0;
    for (long p = static_cast<long>(warp) * SEG; p < n; p += ROUND) mine += load_seg(refs, n, p, &s);
    __syncthreads();
    if (lane == 0) tmp[warp] = mine;
    __syncthreads();
    return __reduce_add_sync(FULL, tmp[lane]);
}

// Calls f(page, free, rank) for every page, rank = how many free pages lie below it; returns the number of free pages.
// Every thread of the CTA takes part; tmp: 32 words of shared memory.
template <typename F>
__device__ __forceinline__ int scan_free(const int32_t* refs, int n, int* tmp, F f) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int base = 0;
    for (long p0 = 0; p0 < n; p0 += ROUND) {
        Seg s;
        const int mine = load_seg(refs, n, p0 + warp * SEG, &s);
        __syncthreads();
        if (lane == 0) tmp[warp] = mine;
        __syncthreads();
        int t = tmp[lane];
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int u = __shfl_up_sync(FULL, t, d);
            if (lane >= d) t += u;
        }
        int rank = base + __shfl_sync(FULL, t, (warp + 31) & 31) * (warp > 0);
        base += __shfl_sync(FULL, t, 31);
#pragma unroll
        for (int u = 0; u < 8; u++) {
            const int c = zeros(s.r[u]);
            int before = c;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int x = __shfl_up_sync(FULL, before, d);
                if (lane >= d) before += x;
            }
            int at = rank + before - c;
            rank += __shfl_sync(FULL, before, 31);
            const long p = s.first + u * 128 + lane * 4;
            const int rr[4] = {s.r[u].x, s.r[u].y, s.r[u].z, s.r[u].w};
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (p + e < n) f(static_cast<int>(p + e), rr[e] == 0, at);
                at += rr[e] == 0;
            }
        }
    }
    return base;
}

// ------------------------------------------------------------------------------------------------ free
// One CTA per listed slot. An entry is claimed by exchange, so a slot named twice is released once.
__global__ void __launch_bounds__(256) k_kv_free(const kx_kv c, const int32_t* seqs, int* status) {
    kx::griddep_wait();
    kx::griddep_launch_dependents();
    const int s = seqs[blockIdx.x];
    if (s < 0) return;
    if (s >= c.n_seqs) {
        if (threadIdx.x == 0) kx::kv_report(status, KX_STATUS_BAD_REQUEST);
        return;
    }
    int32_t* row = c.table + static_cast<long>(s) * c.max_pages;
    for (int j = threadIdx.x; j < c.max_pages; j += blockDim.x) {
        if (__ldcg(row + j) == -1) continue;
        const int p = atomicExch(row + j, -1);
        if (p >= 0 && p < c.n_pages) atomicSub(c.refs + p, 1);
    }
    if (threadIdx.x == 0) c.lens[s] = 0;
}

// ------------------------------------------------------------------------------------------------ extend
struct ExtendWs {
    long long* upto;  // per slot: the pages asked for by the slots up to this one
    int32_t* list;    // the free pages, lowest first, as far as they are asked for
    int32_t* n_free;
};

__device__ __forceinline__ int pages_of(long tokens, int page) { return static_cast<int>((tokens + page - 1) >> (31 - __clz(page))); }

__global__ void __launch_bounds__(PLAN) k_kv_extend_plan(const kx_kv c, const int32_t* want, const ExtendWs w) {
    __shared__ long long tmp[32];
    __shared__ int tmp_i[32];
    kx::griddep_wait();
    kx::griddep_launch_dependents();
    const int tid = threadIdx.x;
    const long cap = static_cast<long>(c.max_pages) * c.page;
    long long base = 0;
    for (int s0 = 0; s0 < c.n_seqs; s0 += PLAN) {
        const int s = s0 + tid;
        int need = 0;
        if (s < c.n_seqs) {
            const int more = want[s], len = c.lens[s];
            if (more > 0 && len >= 0 && len + static_cast<long>(more) <= cap)
                need = pages_of(len + static_cast<long>(more), c.page) - pages_of(len, c.page);
        }
        long long total;
        const long long incl = base + block_scan(need, tmp, &total);
        if (s < c.n_seqs) w.upto[s] = incl;
        base += total;
    }
    const long long asked = base;
    const int n_free = scan_free(c.refs, c.n_pages, tmp_i, [&](int p, bool free, int rank) {
        if (free && rank < asked) w.list[rank] = p;
    });
    if (tid == 0) *w.n_free = n_free;
}

// a warp per slot
__global__ void __launch_bounds__(128) k_kv_extend_take(const kx_kv c, const int32_t* want, int32_t* granted, const ExtendWs w, int* status) {
    const int lane = threadIdx.x & 31;
    const long cap = static_cast<long>(c.max_pages) * c.page;
    kx::griddep_wait();
    kx::griddep_launch_dependents();
    const int s = blockIdx.x * 4 + (threadIdx.x >> 5);
    if (s >= c.n_seqs) return;
    const int more = want[s], len = c.lens[s], n_free = __ldcg(w.n_free);
    const long long last = __ldcg(w.upto + s);
    int grant = 0;
    if (more > 0) {
        if (len < 0 || len > cap) {
            if (lane == 0) kx::kv_report(status, KX_STATUS_BAD_REQUEST);
        } else if (len + static_cast<long>(more) > cap) {
            if (lane == 0) kx::kv_report(status, KX_STATUS_NO_PAGES);
        } else {
            const int have = pages_of(len, c.page), need = pages_of(len + static_cast<long>(more), c.page) - have;
            if (need == 0 || last <= n_free) {
                grant = more;
                int32_t* row = c.table + static_cast<long>(s) * c.max_pages + have;
#pragma unroll 4
                for (int j = lane; j < need; j += 32) {
                    const int p = __ldcg(w.list + (last - need + j));
                    row[j] = p;
                    c.refs[p] = 1;
                }
            } else if (lane == 0) {
                kx::kv_report(status, KX_STATUS_NO_PAGES);
            }
        }
    }
    __syncwarp();  // every lane has read want[s] and lens[s]
    if (lane == 0) {
        granted[s] = grant;
        if (grant) c.lens[s] = len + grant;
    }
}

// ------------------------------------------------------------------------------------------------ append
template <int TYPE, bool VEC>
__device__ __forceinline__ uint4 kv_pack(const float* x) {
    constexpr int E = TYPE == KX_KV_F32 ? 4 : 8;
    float f[E];
    if (VEC) {
#pragma unroll
        for (int e = 0; e < E; e += 4) *reinterpret_cast<float4*>(f + e) = __ldcs(reinterpret_cast<const float4*>(x + e));
    } else {
#pragma unroll
        for (int e = 0; e < E; e++) f[e] = __ldcs(x + e);
    }
    uint4 o;
    uint32_t* w = &o.x;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (TYPE == KX_KV_F32) {
            w[i] = __float_as_uint(f[i]);
        } else if constexpr (TYPE == KX_KV_F16) {
            const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
            const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
    }
    return o;
}

// CTA (s, y): rows y * rb .. of slot s. A thread keeps its place in the rows (16 bytes of the cache; 2^lanes threads per
// row) and goes down them, so that a row costs it a page lookup and two additions: with a place of its own for each 16
// bytes (three divisions) 12 ragged prompts of up to 1999 rows took 20.7 us of GPU time (27.4 from memory), this 19.1 (26.4). HBM-bound: the fp32 rows are read once
// (streaming loads), the narrower rows written once.
template <int TYPE, bool VEC>
__global__ void __launch_bounds__(256) k_kv_append(const kx_kv c, const float* k, int ldk, const float* v, int ldv, const int32_t* count,
                                                   int rows, int rb, int lanes, long k_off, long v_off, int* status) {
    constexpr int E = TYPE == KX_KV_F32 ? 4 : 8, SZ = 16 / E;
    const int s = blockIdx.x, i0 = blockIdx.y * rb;
    kx::griddep_wait();
    kx::griddep_launch_dependents();
    int n = count[s];
    const int len = c.lens[s];
    if (n <= 0) return;
    if (n > rows || n > len || len > static_cast<long>(c.max_pages) * c.page) {  // refused as a whole
        if (threadIdx.x == 0 && blockIdx.y == 0) kx::kv_report(status, KX_STATUS_BAD_REQUEST);
        return;
    }
    if (i0 >= n) return;
    const int first = len - n + i0;  // position of row i0
    n = min(rb, n - i0);
    const int ck = c.heads * (c.dk / E), chunks = ck + c.heads * (c.dv / E);
    const int shift = 31 - __clz(c.page);
    const int32_t* row = c.table + static_cast<long>(s) * c.max_pages;
    for (int x = threadIdx.x & ((1 << lanes) - 1); x < chunks; x += 1 << lanes) {
        const bool isk = x < ck;
        const int per = (isk ? c.dk : c.dv) / E, y = isk ? x : x - ck, h = y / per, d = y - h * per;
        const int ld = isk ? ldk : ldv;
        const float* src = (isk ? k : v) + (static_cast<long>(s) * rows + i0) * ld + y * E;
        char* dst = (isk ? static_cast<char*>(c.k) + k_off : static_cast<char*>(c.v) + v_off) + (static_cast<long>(h) * c.page * per + d) * 16;
        const long page_bytes = (isk ? c.k_page : c.v_page) * SZ;
#pragma unroll 4
        for (int i = threadIdx.x >> lanes; i < n; i += 256 >> lanes) {
            const int pos = first + i, p = row[pos >> shift];
            if (p < 0 || p >= c.n_pages) {
                kx::kv_report(status, KX_STATUS_BAD_REQUEST);
                continue;
            }
            *reinterpret_cast<uint4*>(dst + p * page_bytes + static_cast<long>(pos & (c.page - 1)) * per * 16) =
                kv_pack<TYPE, VEC>(src + static_cast<long>(i) * ld);
        }
    }
}

// ------------------------------------------------------------------------------------------------ moving pages
// The pages from[i] (LAST_FIRST: from[n - 1 - i]) of every layer to the pages to[i], i < n, -1 = none: 16 KB pieces over the grid, four 16-byte loads in flight a
// thread. Sources and targets are different pages.
constexpr int PIECE = 16384;
struct MoveArgs {
    char *k, *v;
    long k_page, k_layer, v_page, v_layer;  // bytes
    int k_bytes, v_bytes, layers;
};

template <bool LAST_FIRST>
__device__ __forceinline__ void move_pages(const MoveArgs& m, const int32_t* from, const int32_t* to, int n) {
    const int ck = (m.k_bytes + PIECE - 1) / PIECE, cv = (m.v_bytes + PIECE - 1) / PIECE, per = (ck + cv) * m.layers;
    for (long t = blockIdx.x; t < static_cast<long>(n) * per; t += gridDim.x) {
        const int i = static_cast<int>(t / per);
        int x = static_cast<int>(t - static_cast<long>(i) * per);
        const int a = from[LAST_FIRST ? n - 1 - i : i], b = to[i];
        if (a < 0 || b < 0) continue;
        const int layer = x / (ck + cv);
        x -= layer * (ck + cv);
        const bool isk = x < ck;
        const int off = (isk ? x : x - ck) * PIECE, left = (isk ? m.k_bytes : m.v_bytes) - off;
        char* base = isk ? m.k + layer * m.k_layer + off : m.v + layer * m.v_layer + off;
        const long st = isk ? m.k_page : m.v_page;
        const char* src = base + a * st;
        char* dst = base + b * st;
        uint4 r[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int o = (u * 256 + threadIdx.x) * 16;
            if (o < left) r[u] = __ldcs(reinterpret_cast<const uint4*>(src + o));
        }
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int o = (u * 256 + threadIdx.x) * 16;
            if (o < left) __stcs(reinterpret_cast<uint4*>(dst + o), r[u]);
        }
    }
}

MoveArgs move_args(const kx_kv* c) {
    const long sz = kx::kv_elem_bytes(c->type);
    MoveArgs m;
    m.k = static_cast<char*>(c->k);
    m.v = static_cast<char*>(c->v);
    m.k_page = c->k_page * sz;
    m.v_page = c->v_page * sz;
    m.k_layer = c->layers > 1 ? c->k_layer * sz : 0;
    m.v_layer = c->layers > 1 ? c->v_layer * sz : 0;
    m.k_bytes = static_cast<int>(c->heads * sz * c->page * c->dk);
    m.v_bytes = static_cast<int>(c->heads * sz * c->page * c->dv);
    m.layers = c->layers;
    return m;
}

// ------------------------------------------------------------------------------------------------ fork
struct ForkWs {
    int32_t *list, *claim, *len, *from, *to;  // free pages; per slot the first pair that names it; per pair its length
                                              // (-1: refused) and the page copied, -1 where none is
};

__global__ void __launch_bounds__(PLAN) k_kv_fork_plan(const kx_kv c, const int32_t* src, const int32_t* dst, int n, const ForkWs w, int* status) {
    __shared__ long long tmp[32];
    __shared__ int tmp_i[32];
    kx::griddep_wait();
    kx::griddep_launch_dependents();
    const int tid = threadIdx.x;
    const long cap = static_cast<long>(c.max_pages) * c.page;
    const int shift = 31 - __clz(c.page);
    const auto slot_ok = [&](int s) { return s >= 0 && s < c.n_seqs; };
    for (int i = tid; i < n; i += PLAN)
        if (slot_ok(dst[i])) w.claim[dst[i]] = INT_MAX;
    __syncthreads();
    for (int i = tid; i < n; i += PLAN)
        if (slot_ok(dst[i])) atomicMin(w.claim + dst[i], i);
    __syncthreads();
    long long base = 0;
    for (int i0 = 0; i0 < n; i0 += PLAN) {
        const int i = i0 + tid;
        int need = 0, len = -1, tail = -1;
        if (i < n && dst[i] >= 0) {
            const int a = src[i], b = dst[i];
            const bool ok = slot_ok(a) && slot_ok(b) && a != b && __ldcg(w.claim + b) == i && c.lens[b] == 0 && c.lens[a] >= 0 &&
                            c.lens[a] <= cap;
            if (ok) {
                len = c.lens[a];
                if (len & (c.page - 1)) {
                    tail = c.table[static_cast<long>(a) * c.max_pages + (len >> shift)];
                    if (tail < 0 || tail >= c.n_pages) {
                        tail = -1;
                        kx::kv_report(status, KX_STATUS_BAD_REQUEST);
                    }
                }
                need = tail >= 0;
            } else {
                kx::kv_report(status, KX_STATUS_BAD_REQUEST);
            }
        }
        long long total;
        const long long incl = base + block_scan(need, tmp, &total);
        if (i < n) {
            w.len[i] = len;
            w.from[i] = tail;
            w.to[i] = need ? static_cast<int>(incl - 1) : -1;  // which free page, for now
        }
        base += total;
    }
    const long long asked = base;
    const int n_free = scan_free(c.refs, c.n_pages, tmp_i, [&](int p, bool free, int rank) {
        if (free && rank < asked) w.list[rank] = p;
    });
    __syncthreads();  // every length has been read before one is written, and the list is there
    for (int i = tid; i < n; i += PLAN) {
        const int len = w.len[i], r = w.to[i];
        if (len < 0) continue;
        if (r >= n_free) {
            w.len[i] = -1;
            w.to[i] = -1;
            kx::kv_report(status, KX_STATUS_NO_PAGES);
            continue;
        }
        if (r >= 0) {
            const int p = w.list[r];
            w.to[i] = p;
            c.refs[p] = 1;
        }
        c.lens[dst[i]] = len;
    }
}

__global__ void __launch_bounds__(256) k_kv_fork_move(const kx_kv c, const int32_t* src, const int32_t* dst, int n, const ForkWs w, const MoveArgs m,
                                                      int* status) {
    kx::griddep_wait();
    kx::griddep_launch_dependents();
    const int shift = 31 - __clz(c.page);
    for (int i = blockIdx.x; i < n; i += gridDim.x) {  // the children's table rows
        const int len = __ldcg(w.len + i);
        if (len < 0) continue;
        const int full = len >> shift, fresh = __ldcg(w.to + i);
        const int32_t* a = c.table + static_cast<long>(src[i]) * c.max_pages;
        int32_t* b = c.table + static_cast<long>(dst[i]) * c.max_pages;
        for (int j = threadIdx.x; j < c.max_pages; j += 256) {
            int p = -1;
            if (j < full) {
                p = a[j];
                if (p >= 0 && p < c.n_pages) {
                    atomicAdd(c.refs + p, 1);
                } else {
                    p = -1;
                    kx::kv_report(status, KX_STATUS_BAD_REQUEST);
                }
            } else if (j == full) {
                p = fresh;
            }
            b[j] = p;
        }
    }
    move_pages<false>(m, w.from, w.to, n);
}

// ------------------------------------------------------------------------------------------------ compact
struct CompactWs {
    int32_t *count, *holes, *late, *map;  // how many pages move; targets; sources, last first; per page its new id
};

// With f(p) free pages below p: a free page p < n_live is hole f(p); a live page p has p - f(p) live pages below it, so
// among the live pages from n_live on it is the (n_live - 1 - (p - f(p)))-th from the end.
__global__ void __launch_bounds__(PLAN) k_kv_compact_plan(const kx_kv c, const CompactWs w, int32_t* n_live_out) {
    __shared__ int tmp_i[32];
    __shared__ int n_late;
    kx::griddep_wait();
    kx::griddep_launch_dependents();
    const int tid = threadIdx.x;
    if (tid == 0) n_late = 0;
    const int n_live = c.n_pages - count_free(c.refs, c.n_pages, tmp_i);
    int mine = 0;
    scan_free(c.refs, c.n_pages, tmp_i, [&](int p, bool free, int rank) {
        if (p < n_live) {
            if (free) w.holes[rank] = p;
        } else if (!free) {
            w.late[n_live - 1 - (p - rank)] = p;
            mine++;
        } else {
            w.map[p] = p;
        }
    });
    mine = __reduce_add_sync(FULL, mine);
    if ((tid & 31) == 0) atomicAdd(&n_late, mine);
    __syncthreads();
    for (int r = tid; r < n_late; r += PLAN) {
        const int to = w.holes[r], from = w.late[n_late - 1 - r];
        w.map[from] = to;
        c.refs[to] = c.refs[from];
        c.refs[from] = 0;
    }
    if (tid == 0) {
        *w.count = n_late;
        *n_live_out = n_live;
    }
}

__global__ void __launch_bounds__(256) k_kv_compact_move(const kx_kv c, const CompactWs w, const int32_t* n_live_p,
                                                         const MoveArgs m) {
    kx::griddep_wait();
    kx::griddep_launch_dependents();
    const int n_late = __ldcg(w.count), n_live = __ldcg(n_live_p);
    if (n_late == 0) return;
    const long entries = static_cast<long>(c.n_seqs) * c.max_pages;
    for (long i = blockIdx.x * 256l + threadIdx.x; i < entries; i += gridDim.x * 256l) {
        const int p = c.table[i];
        if (p >= n_live && p < c.n_pages) c.table[i] = __ldcg(w.map + p);
    }
    move_pages<true>(m, w.late, w.holes, n_late);
}

int sm_count() {
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0)
        sms = 148;
    return sms;
}

bool ws_ok(const kx_kv* c, const void* ws, size_t ws_bytes) {
    return kx::kv_ok(c) && ws && (reinterpret_cast<uintptr_t>(ws) & 15) == 0 && ws_bytes >= kx_kv_ws(c);
}

}  // namespace

extern "C" {

// the largest of: extend (list, 8-byte sums per slot), fork (list, four words per slot), compact (three lists, a count)
size_t kx_kv_ws(const kx_kv* c) {
    if (!kx::kv_ok(c)) return 0;
    const size_t pages = (static_cast<size_t>(c->n_pages) + 3) / 4 * 4;
    return 4 * (3 * pages + 4 * static_cast<size_t>(c->n_seqs) + 16);
}

int kx_kv_free(const kx_kv* c, const int32_t* seqs, int n, int* status, void* stream) {
    if (!kx::kv_ok(c) || n < 0) return -1;
    if (n == 0) return 0;
    if (!seqs) return -1;
    return kx::launch_pdl(k_kv_free, dim3(n), dim3(256), 0, static_cast<cudaStream_t>(stream), *c, seqs, status);
}

int kx_kv_extend(const kx_kv* c, const int32_t* want, int32_t* granted, void* ws, size_t ws_bytes, int* status, void* stream) {
    if (!ws_ok(c, ws, ws_bytes) || !want || !granted) return -1;
    ExtendWs w;
    w.upto = static_cast<long long*>(ws);
    w.n_free = reinterpret_cast<int32_t*>(w.upto + c->n_seqs);
    w.list = w.n_free + 4;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (kx::launch_pdl(k_kv_extend_plan, dim3(1), dim3(PLAN), 0, st, *c, want, w) != 0) return -1;
    return kx::launch_pdl(k_kv_extend_take, dim3((c->n_seqs + 3) / 4), dim3(128), 0, st, *c, want, granted, w, status);
}

int kx_kv_append(const kx_kv* c, int layer, const float* k, int ldk, const float* v, int ldv, const int32_t* count, int rows,
                 int* status, void* stream) {
    if (!kx::kv_ok(c) || layer < 0 || layer >= c->layers || rows < 0) return -1;
    if (rows == 0) return 0;
    if (!k || !v || !count || ldk < c->heads * c->dk || ldv < c->heads * c->dv) return -1;
    const int chunks = c->heads * (c->dk + c->dv) / (16 / static_cast<int>(kx::kv_elem_bytes(c->type)));
    int lanes = 0;
    while (lanes < 8 && 1 << lanes < chunks) lanes++;
    // 16 rows per thread, 65535 CTAs per slot at most
    const int rb = std::max(16 << (8 - lanes), (rows - 1) / 65535 + 1);
    const dim3 grid(c->n_seqs, (rows - 1) / rb + 1);
    const bool vec = ((ldk | ldv) & 3) == 0 && ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0;
    const long sz = kx::kv_elem_bytes(c->type);
    const long k_off = layer ? layer * c->k_layer * sz : 0, v_off = layer ? layer * c->v_layer * sz : 0;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const auto launch = [&](auto kernel) {
        return kx::launch_pdl(kernel, grid, dim3(256), 0, st, *c, k, ldk, v, ldv, count, rows, rb, lanes, k_off, v_off, status);
    };
    if (c->type == KX_KV_F32) return vec ? launch(k_kv_append<KX_KV_F32, true>) : launch(k_kv_append<KX_KV_F32, false>);
    if (c->type == KX_KV_F16) return vec ? launch(k_kv_append<KX_KV_F16, true>) : launch(k_kv_append<KX_KV_F16, false>);
    return vec ? launch(k_kv_append<KX_KV_BF16, true>) : launch(k_kv_append<KX_KV_BF16, false>);
}

int kx_kv_fork(const kx_kv* c, const int32_t* src, const int32_t* dst, int n, void* ws, size_t ws_bytes, int* status, void* stream) {
    if (!ws_ok(c, ws, ws_bytes) || n < 0 || n > c->n_seqs) return -1;
    if (n == 0) return 0;
    if (!src || !dst) return -1;
    ForkWs w;
    w.list = static_cast<int32_t*>(ws);
    w.claim = w.list + (c->n_pages + 3) / 4 * 4;
    w.len = w.claim + c->n_seqs;
    w.from = w.len + c->n_seqs;
    w.to = w.from + c->n_seqs;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (kx::launch_pdl(k_kv_fork_plan, dim3(1), dim3(PLAN), 0, st, *c, src, dst, n, w, status) != 0) return -1;
    return kx::launch_pdl(k_kv_fork_move, dim3(sm_count() * 4), dim3(256), 0, st, *c, src, dst, n, w, move_args(c), status);
}

int kx_kv_compact(const kx_kv* c, int32_t* n_live, void* ws, size_t ws_bytes, void* stream) {
    if (!ws_ok(c, ws, ws_bytes) || !n_live) return -1;
    CompactWs w;
    const size_t pages = (static_cast<size_t>(c->n_pages) + 3) / 4 * 4;
    w.holes = static_cast<int32_t*>(ws);
    w.late = w.holes + pages;
    w.map = w.late + pages;
    w.count = w.map + pages;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (kx::launch_pdl(k_kv_compact_plan, dim3(1), dim3(PLAN), 0, st, *c, w, n_live) != 0) return -1;
    return kx::launch_pdl(k_kv_compact_move, dim3(sm_count() * 8), dim3(256), 0, st, *c, w, static_cast<const int32_t*>(n_live), move_args(c));
}

}  // extern "C"
