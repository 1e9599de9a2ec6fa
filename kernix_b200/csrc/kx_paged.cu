// KERNIX-B200 attention of one new token per sequence over a paged key-value cache (kx_attention_paged,
// include/kx_kernels.h). Per row and query head, over the keys j that the token at position len - 1 sees:
//   ctx = sum_j p_j v_j / sum_j p_j,  p_j = exp(s_j - max s),  s_j = scale q.k_j.
//
// Bound: HBM, each visible key and value row read once for all the query heads that share it. Design:
//   * The keys of a (row, key-value head) are walked in steps of 16 (8 for an fp32 cache), aligned in the sequence.
//     A warp takes a step at a time on its own: running maximum, sum and output in registers, no barrier until the end.
//   * Both products run as mma.sync with up to 8 query heads as the rows 0-7 of a 16-row tile, so that 8 heads cost the
//     CUDA cores no more than one would (plain multiplies in fp32 would be as long as the loads from 4 heads per
//     key-value head on). The cache's elements enter exactly as they are stored; the fp32 side (q, then p) is split into
//     parts of the cache's type, whose products land in rows 0-7 (part 1) and 8-15 (part 2) of the same tile:
//       f16:  2 parts of 11 bits, q scaled by a power of two per head to use f16's range, p in [0, 2^13];
//       bf16: 3 parts of 8 bits, the third as a second product;
//       f32:  tf32 halves, q.k = qh.kh + ql.kh + qh.kl (and p.v likewise), 11 + 11 bits.
//     That keeps fp32's accuracy (parts lost: below 2^-22 of the operand). A step's p.v is added to the output in
//     fp32 registers by CUDA-core adds, not carried through the tensor core's truncating accumulation.
//   * Loads: every lane copies (cp.async, 16 bytes) exactly the chunks that it will use itself as matrix fragments, into
//     a ring of its own in shared memory: deep prefetch without registers and without barriers. The order of the
//     reduction axis inside a product is free, so a lane's 16 contiguous bytes serve as they lie; masked keys are
//     zero-filled and never read.
//   * Work split: the steps of all rows and heads form one line, cut into equal ranges, one per CTA (two CTAs per SM);
//     a range may cover several short sequences or a part of a long one. A head whose steps lie in several ranges is
//     joined by a second launch (programmatic dependent) in the order of the ranges: nothing depends on timing.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "kx_kernels.h"
#include "kx_kv.cuh"
#include "kx_pdl.cuh"
#include "kx_sm100.cuh"

namespace kx {
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
}  // namespace kx

namespace {

constexpr unsigned FULL = 0xFFFFFFFFu;
constexpr int PG_WARPS = 4, PG_THREADS = PG_WARPS * 32;
constexpr int PG_STAGES = 3;
constexpr int PG_HEADS = 8;       // query heads per tile
constexpr int PG_MAX_CTAS = 512;  // of a split launch: sizes the workspace
constexpr int PG_MIN_STEPS = 4 * PG_WARPS;  // a CTA's range is at least this many steps: the join costs as much as a few
constexpr int PG_DMAX = 128;

struct PagedArgs {
    kx_kv c;
    const char *k, *v;  // the layer's pools
    const float* q;
    float* ctx;
    const int32_t* seqs;
    char* ws;
    int* status;
    int n, H, G, chunks, per_chunk;  // query heads per key-value head, tiles of heads per key-value head, heads per tile
    int ldq, ldc, window, sinks, grid;
    float scale2;
    bool vecq;
};

// what a CTA's range begins with: written by the main launch, read by the join
struct PagedDesc {
    long long first;  // position of the unit's first step on the line
    long long per;    // steps per CTA
    int row, unit, steps, pad;
};

// the steps of a row's token: the steps that hold its first tokens, then those of its window
struct Span {
    int len, s0, w0;    // visible: j < s0 or w0 <= j < len
    int na, b0, steps;  // steps 0 .. na - 1, then b0, b0 + 1, ...
    bool bad;           // the row's slot or length is out of range
};
template <int KS>
__device__ __forceinline__ Span span_of(const PagedArgs& A, int row, int* slot) {
    Span sp;
    const int s = A.seqs ? A.seqs[row] : row;
    *slot = s;
    if (s < 0) {
        sp = Span{0, 0, 0, 0, 0, 0, false};
        return sp;
    }
    int len = s < A.c.n_seqs ? A.c.lens[s] : -1;
    sp.bad = len < 0 || len > static_cast<long>(A.c.max_pages) * A.c.page;
    if (sp.bad) len = 0;
    sp.len = len;
    sp.w0 = A.window > 0 && len > A.window ? len - A.window : 0;
    sp.s0 = min(A.sinks, sp.w0);
    sp.na = (sp.s0 + KS - 1) / KS;
    sp.b0 = max(sp.na, sp.w0 / KS);
    sp.steps = max(1, sp.na + (len + KS - 1) / KS - sp.b0);  // a row that sees nothing still has its zeros to write
    return sp;
}

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool ok) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t a) {
    uint4 r;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(a) : "memory");
    return r;
}

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// two fp32 values as PARTS pairs of the 16-bit type, the value = the sum of its parts up to the last one's rounding
template <int TYPE>
__device__ __forceinline__ uint32_t pack2(float a, float b, float* ra, float* rb) {
    uint32_t w;
    if constexpr (TYPE == KX_KV_F16) {
        const __half2 h = __floats2half2_rn(a, b);
        const float2 f = __half22float2(h);
        *ra = a - f.x;
        *rb = b - f.y;
        w = *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        const float2 f = __bfloat1622float2(h);
        *ra = a - f.x;
        *rb = b - f.y;
        w = *reinterpret_cast<const uint32_t*>(&h);
    }
    return w;
}
__device__ __forceinline__ uint32_t tf32_of(float v, float* rest) {
    float hi, lo;
    kx::tf32_split(v, hi, lo);
    *rest = lo;
    return __float_as_uint(hi);
}

template <int TYPE, int D>
struct Shape {
    static constexpr int EPC = TYPE == KX_KV_F32 ? 4 : 8;   // elements per 16-byte chunk
    static constexpr int KT = TYPE == KX_KV_F32 ? 1 : 2;    // tiles of 8 keys per step
    static constexpr int KS = 8 * KT;                       // keys per step
    static constexpr int KCH = D / EPC / 4;                 // K chunks per lane and tile: chunk 4 c + t of key g
    static constexpr int VK = 2 * KT;                       // V keys per lane: 2 t, 2 t + 1 of each tile
    static constexpr int VCH = D / EPC / 8;                 // V chunks per lane and key: chunk 8 c + g
    static constexpr int CH = KT * KCH + VK * VCH;
    static constexpr int STAGE = CH * 32 * 16;              // bytes per warp and stage
    static constexpr int QW = D / 4;                        // q elements per lane
    static constexpr int PARTS = TYPE == KX_KV_BF16 ? 3 : 2;
    static constexpr int QP = TYPE == KX_KV_F32 ? QW : QW / 2;  // 32-bit words per part
    static constexpr int SMEM = PG_WARPS * PG_STAGES * STAGE;
    static_assert(PG_STAGES * STAGE >= PG_HEADS * D * 4, "a warp's ring holds its partial output");
};

// One unit's steps [i0, i1) (of sp.steps) by the whole CTA. UNSPLIT results go to ctx, others to `part`.
template <int TYPE, int D>
__device__ void paged_piece(const PagedArgs& A, uint8_t* smem, float (&red)[PG_WARPS][PG_HEADS][2], int row, int slot, const Span& sp,
                            int unit, int i0, int i1, float* part) {
    using S = Shape<TYPE, D>;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int kvh = unit / A.chunks, head0 = kvh * A.G + (unit - kvh * A.chunks) * A.per_chunk;
    const int heads = min(A.per_chunk, (kvh + 1) * A.G - head0);
    const int nck = A.c.dk / S::EPC, ncv = A.c.dv / S::EPC, shift = 31 - __clz(A.c.page);
    const int32_t* table = A.c.table + static_cast<long>(slot) * A.c.max_pages;
    constexpr long SZ = 16 / S::EPC;
    const char* kb = A.k + static_cast<long>(kvh) * A.c.page * A.c.dk * SZ;
    const char* vb = A.v + static_cast<long>(kvh) * A.c.page * A.c.dv * SZ;
    const uint32_t ring = kx::smem_u32(smem) + warp * (PG_STAGES * S::STAGE) + lane * 16;
    bool bad = sp.bad;

    const auto first_key = [&](int i) { return (i < sp.na ? i : i - sp.na + sp.b0) * S::KS; };
    const auto visible = [&](int j) { return j < sp.len && (j < sp.s0 || j >= sp.w0); };
    // page of key first_key(i) + lane % KS, one step ahead of its use
    const auto page_of = [&](int i) {
        const int j = first_key(i) + (lane & (S::KS - 1));
        return i < i1 && visible(j) ? __ldg(table + (j >> shift)) : 0;
    };
    const auto issue = [&](int i, int pid, int stage) {
        if (i < i1) {
            const int base = first_key(i);
            if (pid < 0 || pid >= A.c.n_pages) {
                bad = true;  // this key's page is not there: the row becomes NaN, nothing is read
                pid = -1;
            }
            const uint32_t dst = ring + stage * S::STAGE;
#pragma unroll
            for (int u = 0; u < S::KT; u++) {
                const int j = base + u * 8 + g, p = __shfl_sync(FULL, pid, u * 8 + g);
                const bool ok = visible(j) && p >= 0;
                const char* src = ok ? kb + p * A.c.k_page * SZ + (static_cast<long>(j & (A.c.page - 1)) * nck + t) * 16 : A.k;
#pragma unroll
                for (int c = 0; c < S::KCH; c++) {
                    const bool in = ok && c * 4 + t < nck;
                    if (c * 4 < nck) cp16(dst + (u * S::KCH + c) * 512, in ? src + c * 64 : A.k, in);
                }
            }
#pragma unroll
            for (int u = 0; u < S::VK; u++) {
                const int x = (u >> 1) * 8 + 2 * t + (u & 1), j = base + x, p = __shfl_sync(FULL, pid, x);
                const bool ok = visible(j) && p >= 0;
                const char* src = ok ? vb + p * A.c.v_page * SZ + (static_cast<long>(j & (A.c.page - 1)) * ncv + g) * 16 : A.v;
#pragma unroll
                for (int c = 0; c < S::VCH; c++) {
                    const bool in = ok && c * 8 + g < ncv;
                    if (c * 8 < ncv) cp16(dst + (S::KT * S::KCH + u * S::VCH + c) * 512, in ? src + c * 128 : A.v, in);
                }
            }
        }
        cp_commit();
    };

    // the first stages on their way before q is looked at
    int pid = page_of(i0 + warp);
#pragma unroll
    for (int s = 0; s < PG_STAGES - 1; s++) {
        const int next = page_of(i0 + warp + (s + 1) * PG_WARPS);
        issue(i0 + warp + s * PG_WARPS, pid, s);
        pid = next;
    }

    // q of head g: lane t holds the elements that its K chunks hold
    uint32_t qp[S::PARTS][S::QP];
    float qscale = A.scale2, off = 0.0f;
    {
        float x[S::QW];
        const float* qr = A.q + static_cast<long>(row) * A.ldq + static_cast<long>(head0 + min(g, heads - 1)) * A.c.dk;
#pragma unroll
        for (int c = 0; c < S::KCH; c++)
#pragma unroll
            for (int e = 0; e < S::EPC; e += 4) {
                const int d = (c * 4 + t) * S::EPC + e;
                float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
                if (d < A.c.dk) f = A.vecq ? *reinterpret_cast<const float4*>(qr + d) : make_float4(qr[d], qr[d + 1], qr[d + 2], qr[d + 3]);
                x[c * S::EPC + e] = f.x;
                x[c * S::EPC + e + 1] = f.y;
                x[c * S::EPC + e + 2] = f.z;
                x[c * S::EPC + e + 3] = f.w;
            }
        if constexpr (TYPE == KX_KV_F16) {
            // |q| < 2^14 after the scaling; parts keep 22 bits of what is above 2^-17 of the head's largest element
            float m = 0.0f;
#pragma unroll
            for (int i = 0; i < S::QW; i++) m = fmaxf(m, fabsf(x[i]));
            m = fmaxf(m, __shfl_xor_sync(FULL, m, 1));
            m = fmaxf(m, __shfl_xor_sync(FULL, m, 2));
            const int e = min(max(static_cast<int>(__float_as_uint(m) >> 23) - 127, -100), 126);  // floor(log2 m)
            const float up = __uint_as_float(static_cast<uint32_t>(127 + 13 - e) << 23);
            qscale *= __uint_as_float(static_cast<uint32_t>(127 - 13 + e) << 23);
            off = 13.0f;
#pragma unroll
            for (int i = 0; i < S::QW; i++) x[i] *= up;
        }
        if constexpr (TYPE == KX_KV_F32) {
#pragma unroll
            for (int i = 0; i < S::QW; i++) {
                float lo;
                qp[0][i] = tf32_of(x[i], &lo);
                qp[1][i] = __float_as_uint(lo);
            }
        } else {
#pragma unroll
            for (int i = 0; i < S::QP; i++) {
                float a = x[2 * i], b = x[2 * i + 1];
#pragma unroll
                for (int p = 0; p < S::PARTS; p++) qp[p][i] = pack2<TYPE>(a, b, &a, &b);
            }
        }
    }

    float o[D / 4];
#pragma unroll
    for (int i = 0; i < D / 4; i++) o[i] = 0.0f;
    float m = -INFINITY, l = 0.0f;
    int stage = 0;
    for (int i = i0 + warp; i < i1; i += PG_WARPS) {
        {
            const int ahead = i + (PG_STAGES - 1) * PG_WARPS;
            const int next = page_of(ahead + PG_WARPS);
            issue(ahead, pid, stage == 0 ? PG_STAGES - 1 : stage - 1);
            pid = next;
        }
        cp_wait<PG_STAGES - 1>();
        const uint32_t src = ring + stage * S::STAGE;
        stage = stage + 1 == PG_STAGES ? 0 : stage + 1;

        // scores: rows 0-7 and 8-15 of the tile are the products of q's parts
        float s[2 * S::KT];
#pragma unroll
        for (int u = 0; u < S::KT; u++) {
            float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < S::KCH; c++) {
                if (c * 4 >= nck) continue;
                const uint4 kv = lds16(src + (u * S::KCH + c) * 512);
                if constexpr (TYPE == KX_KV_F32) {
                    const uint32_t w[4] = {kv.x, kv.y, kv.z, kv.w};
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const int x = c * 4 + 2 * h;
                        float l0, l1;
                        const uint32_t h0 = tf32_of(__uint_as_float(w[2 * h]), &l0), h1 = tf32_of(__uint_as_float(w[2 * h + 1]), &l1);
                        mma_tf32(d, qp[0][x], qp[1][x], qp[0][x + 1], qp[1][x + 1], h0, h1);
                        mma_tf32(d, qp[0][x], 0, qp[0][x + 1], 0, __float_as_uint(l0), __float_as_uint(l1));
                    }
                } else {
                    const int x = c * 4;
                    if constexpr (TYPE == KX_KV_F16) {
                        mma_f16(d, qp[0][x], qp[1][x], qp[0][x + 1], qp[1][x + 1], kv.x, kv.y);
                        mma_f16(d, qp[0][x + 2], qp[1][x + 2], qp[0][x + 3], qp[1][x + 3], kv.z, kv.w);
                    } else {
                        mma_bf16(d, qp[0][x], qp[1][x], qp[0][x + 1], qp[1][x + 1], kv.x, kv.y);
                        mma_bf16(d, qp[0][x + 2], qp[1][x + 2], qp[0][x + 3], qp[1][x + 3], kv.z, kv.w);
                        mma_bf16(d, qp[2][x], 0, qp[2][x + 1], 0, kv.x, kv.y);
                        mma_bf16(d, qp[2][x + 2], 0, qp[2][x + 3], 0, kv.z, kv.w);
                    }
                }
            }
            const int j = first_key(i) + u * 8 + 2 * t;
            s[2 * u] = visible(j) ? (d[0] + d[2]) * qscale : -INFINITY;
            s[2 * u + 1] = visible(j + 1) ? (d[1] + d[3]) * qscale : -INFINITY;
        }
        float mx = s[0];
#pragma unroll
        for (int e = 1; e < 2 * S::KT; e++) mx = fmaxf(mx, s[e]);
        mx = fmaxf(mx, __shfl_xor_sync(FULL, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(FULL, mx, 2));
        const float mn = fmaxf(m, mx);
        const float safe = mn == -INFINITY ? 0.0f : mn;
        if (__any_sync(FULL, mn > m)) {
            const float alpha = kx::ex2(m - safe);
            l *= alpha;
#pragma unroll
            for (int e = 0; e < D / 4; e++) o[e] *= alpha;
        }
        m = mn;
        float p[2 * S::KT];
#pragma unroll
        for (int e = 0; e < 2 * S::KT; e++) {
            p[e] = kx::ex2(s[e] - (safe - off));
            l += p[e];
        }

        // p.v: column 2 t (2 t + 1) of n-tile (c, e) is element e of chunk 8 c + 2 t (+ 1)
        if constexpr (TYPE == KX_KV_F32) {
            float q0, q1;
            const uint32_t h0 = tf32_of(p[0], &q0), h1 = tf32_of(p[1], &q1);
#pragma unroll
            for (int c = 0; c < S::VCH; c++) {
                if (c * 8 >= ncv) continue;
                const uint4 va = lds16(src + (S::KT * S::KCH + c) * 512), vbq = lds16(src + (S::KT * S::KCH + S::VCH + c) * 512);
                const uint32_t wa[4] = {va.x, va.y, va.z, va.w}, wb[4] = {vbq.x, vbq.y, vbq.z, vbq.w};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float d[4] = {0.f, 0.f, 0.f, 0.f}, l0, l1;
                    const uint32_t v0 = tf32_of(__uint_as_float(wa[e]), &l0), v1 = tf32_of(__uint_as_float(wb[e]), &l1);
                    mma_tf32(d, h0, 0, h1, 0, __float_as_uint(l0), __float_as_uint(l1));
                    mma_tf32(d, h0, __float_as_uint(q0), h1, __float_as_uint(q1), v0, v1);
                    o[c * 8 + e] += d[0] + d[2];
                    o[c * 8 + 4 + e] += d[1] + d[3];
                }
            }
        } else {
            uint32_t pa[S::PARTS], pb[S::PARTS];
            {
                float a = p[0], b = p[1], c = p[2], d = p[3];
#pragma unroll
                for (int x = 0; x < S::PARTS; x++) {
                    pa[x] = pack2<TYPE>(a, b, &a, &b);
                    pb[x] = pack2<TYPE>(c, d, &c, &d);
                }
            }
#pragma unroll
            for (int c = 0; c < S::VCH; c++) {
                if (c * 8 >= ncv) continue;
                uint32_t w[4][4];
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const uint4 x = lds16(src + (S::KT * S::KCH + u * S::VCH + c) * 512);
                    w[u][0] = x.x, w[u][1] = x.y, w[u][2] = x.z, w[u][3] = x.w;
                }
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const uint32_t sel = e & 1 ? 0x7632 : 0x5410;
                    const uint32_t b0 = __byte_perm(w[0][e >> 1], w[1][e >> 1], sel), b1 = __byte_perm(w[2][e >> 1], w[3][e >> 1], sel);
                    float d[4] = {0.f, 0.f, 0.f, 0.f};
                    if constexpr (TYPE == KX_KV_F16) {
                        mma_f16(d, pa[0], pa[1], pb[0], pb[1], b0, b1);
                    } else {
                        mma_bf16(d, pa[2], 0, pb[2], 0, b0, b1);
                        mma_bf16(d, pa[0], pa[1], pb[0], pb[1], b0, b1);
                    }
                    o[c * 16 + e] += d[0] + d[2];
                    o[c * 16 + 8 + e] += d[1] + d[3];
                }
            }
        }
    }
    cp_wait<0>();

    // the warps' partial results meet in shared memory (each in the place of its own ring)
    bad = __any_sync(FULL, bad);
    l += __shfl_xor_sync(FULL, l, 1);
    l += __shfl_xor_sync(FULL, l, 2);
    __syncwarp();
    if (t == 0) {
        red[warp][g][0] = m;
        red[warp][g][1] = bad ? NAN : l;
    }
    if (bad && lane == 0) kx::kv_report(A.status, KX_STATUS_BAD_REQUEST);
    float* mine = reinterpret_cast<float*>(smem + warp * (PG_STAGES * S::STAGE));
    // lane (g, t): 2 EPC contiguous elements of head g per V chunk group
#pragma unroll
    for (int c = 0; c < S::VCH; c++)
#pragma unroll
        for (int e = 0; e < 2 * S::EPC; e += 4)
            *reinterpret_cast<float4*>(mine + g * D + c * 8 * S::EPC + t * 2 * S::EPC + e) =
                make_float4(o[c * 2 * S::EPC + e], o[c * 2 * S::EPC + e + 1], o[c * 2 * S::EPC + e + 2], o[c * 2 * S::EPC + e + 3]);
    __syncthreads();
    for (int x = tid; x < heads * D; x += PG_THREADS) {
        const int h = x / D, d = x - h * D;
        float mm = red[0][h][0];
#pragma unroll
        for (int w = 1; w < PG_WARPS; w++) mm = fmaxf(mm, red[w][h][0]);
        const float ms = mm == -INFINITY ? 0.0f : mm;
        float num = 0.0f, den = 0.0f;
#pragma unroll
        for (int w = 0; w < PG_WARPS; w++) {
            const float f = kx::ex2(red[w][h][0] - ms);
            den += f * red[w][h][1];
            num += f * reinterpret_cast<const float*>(smem + w * (PG_STAGES * S::STAGE))[x];
        }
        if (part) {
            part[x] = num;
            if (d == 0) {
                part[PG_HEADS * PG_DMAX + 2 * h] = mm;
                part[PG_HEADS * PG_DMAX + 2 * h + 1] = den;
            }
        } else if (d < A.c.dv) {
            A.ctx[static_cast<long>(row) * A.ldc + static_cast<long>(head0 + h) * A.c.dv + d] = den == 0.0f ? 0.0f : num / den;
        }
    }
    __syncthreads();  // the rings and `red` are free for the next piece
}

constexpr size_t PG_PART = (PG_HEADS * PG_DMAX + 2 * PG_HEADS) * sizeof(float);
__device__ __host__ inline size_t part_offset(int cta, int which) {
    return PG_MAX_CTAS * sizeof(PagedDesc) + (static_cast<size_t>(cta) * 2 + which) * PG_PART;
}

__device__ __forceinline__ long long warp_sum(long long v) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(FULL, v, d);
    return v;
}

// SPLIT: CTA j takes the steps [j per, (j + 1) per) of the line; otherwise CTA j is one unit
template <int TYPE, int D, bool SPLIT>
__global__ void __launch_bounds__(PG_THREADS, 2) k_paged(const PagedArgs A) {
    using S = Shape<TYPE, D>;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float red[PG_WARPS][PG_HEADS][2];
    __shared__ long long sums[PG_WARPS];
    __shared__ long long found_first;
    __shared__ int found_row;
    const int units = A.c.heads * A.chunks, tid = threadIdx.x, lane = tid & 31;
    kx::griddep_wait();
    kx::griddep_launch_dependents();
    int slot;
    if constexpr (!SPLIT) {
        const int row = blockIdx.x / units;
        const Span sp = span_of<S::KS>(A, row, &slot);
        if (slot < 0) return;
        paged_piece<TYPE, D>(A, smem, red, row, slot < A.c.n_seqs ? slot : 0, sp, blockIdx.x - row * units, 0, sp.steps, nullptr);
        return;
    }
    // the line's length, then the row that this CTA's range begins in
    long long mine = 0;
    for (int r = tid; r < A.n; r += PG_THREADS) mine += span_of<S::KS>(A, r, &slot).steps;
    mine = warp_sum(mine);
    if (lane == 0) sums[tid >> 5] = mine;
    if (tid == 0) found_row = -1;
    __syncthreads();
    long long total = 0;
#pragma unroll
    for (int w = 0; w < PG_WARPS; w++) total += sums[w];
    total *= units;
    const long long per = max((total + A.grid - 1) / A.grid, static_cast<long long>(PG_MIN_STEPS));
    const long long lo = blockIdx.x * per, hi = min(lo + per, total);
    PagedDesc* desc = reinterpret_cast<PagedDesc*>(A.ws) + blockIdx.x;
    if (lo >= total) {
        if (tid == 0) desc->row = -1;
        return;
    }
    long long before = 0;
    for (int r0 = 0; r0 < A.n; r0 += PG_THREADS) {
        const int r = r0 + tid;
        const long long st = r < A.n ? static_cast<long long>(span_of<S::KS>(A, r, &slot).steps) * units : 0;
        long long incl = st;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const long long u = __shfl_up_sync(FULL, incl, d);
            if (lane >= d) incl += u;
        }
        __syncthreads();
        if (lane == 31) sums[tid >> 5] = incl;
        __syncthreads();
        long long all = 0;
#pragma unroll
        for (int w = 0; w < PG_WARPS; w++) {
            if (w < (tid >> 5)) incl += sums[w];
            all += sums[w];
        }
        incl += before;
        if (lo < incl && lo >= incl - st) {
            found_row = r;
            found_first = incl - st;
        }
        before += all;
        if (lo < before) break;
    }
    __syncthreads();
    int row = found_row;
    long long first = found_first;  // the row's first step on the line
    for (long long at = lo; at < hi; row++) {
        const Span sp = span_of<S::KS>(A, row, &slot);
        if (slot < 0) continue;
        int unit = static_cast<int>((at - first) / sp.steps);
        for (; unit < units && at < hi; unit++) {
            const long long u0 = first + static_cast<long long>(unit) * sp.steps, u1 = u0 + sp.steps;
            if (at == lo && tid == 0) *desc = PagedDesc{u0, per, row, unit, sp.steps, 0};
            const long long end = min(u1, hi);
            float* part = nullptr;  // a unit in several ranges: its first part in place 1, the others in place 0
            if (at != u0 || end != u1) part = reinterpret_cast<float*>(A.ws + part_offset(blockIdx.x, at == u0));
            paged_piece<TYPE, D>(A, smem, red, row, slot < A.c.n_seqs ? slot : 0, sp, unit, static_cast<int>(at - u0),
                                 static_cast<int>(end - u0), part);
            at = end;
        }
        first += static_cast<long long>(sp.steps) * units;
    }
}

// CTA (j, h): if the range of CTA j + 1 begins inside a unit whose first step lies in the range of CTA j, joins that
// unit's parts for head h, in their order: each warp every 4th part, then the warps.
__global__ void __launch_bounds__(128) k_paged_join(const PagedArgs A) {
    __shared__ float acc[4][PG_DMAX];
    __shared__ float ml[4][2];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, h = blockIdx.y;
    kx::griddep_wait();
    const PagedDesc ds = reinterpret_cast<const PagedDesc*>(A.ws)[blockIdx.x + 1];
    if (ds.row < 0) return;
    const long long j0 = ds.first / ds.per, j1 = (ds.first + ds.steps - 1) / ds.per;
    if (j0 != blockIdx.x || ds.first == (blockIdx.x + 1) * ds.per) return;
    const int kvh = ds.unit / A.chunks, head0 = kvh * A.G + (ds.unit - kvh * A.chunks) * A.per_chunk;
    if (h >= min(A.per_chunk, (kvh + 1) * A.G - head0)) return;
    const int D = A.c.dk <= 64 && A.c.dv <= 64 ? 64 : 128;
    const int d = lane * 4;
    const auto part = [&](long long j) { return reinterpret_cast<const float*>(A.ws + part_offset(static_cast<int>(j), j == j0)); };
    float m = -INFINITY;
    for (long long j = j0 + lane; j <= j1; j += 32) m = fmaxf(m, __ldcg(part(j) + PG_HEADS * PG_DMAX + 2 * h));
#pragma unroll
    for (int x = 16; x; x >>= 1) m = fmaxf(m, __shfl_xor_sync(FULL, m, x));
    const float ms = m == -INFINITY ? 0.0f : m;
    float4 num = make_float4(0.f, 0.f, 0.f, 0.f);
    float den = 0.0f;
#pragma unroll 4
    for (long long j = j0 + warp; j <= j1; j += 4) {
        const float* p = part(j);
        const float2 st = __ldcg(reinterpret_cast<const float2*>(p + PG_HEADS * PG_DMAX + 2 * h));
        const float f = kx::ex2(st.x - ms);
        const float4 v = d < D ? __ldcg(reinterpret_cast<const float4*>(p + h * D + d)) : make_float4(0.f, 0.f, 0.f, 0.f);
        den += f * st.y;
        num.x += f * v.x;
        num.y += f * v.y;
        num.z += f * v.z;
        num.w += f * v.w;
    }
    *reinterpret_cast<float4*>(&acc[warp][d]) = num;
    if (lane == 0) ml[warp][0] = den;
    __syncthreads();
    const int x = threadIdx.x;
    if (x < A.c.dv) {
        const float n = acc[0][x] + acc[1][x] + acc[2][x] + acc[3][x], l = ml[0][0] + ml[1][0] + ml[2][0] + ml[3][0];
        A.ctx[static_cast<long>(ds.row) * A.ldc + static_cast<long>(head0 + h) * A.c.dv + x] = l == 0.0f ? 0.0f : n / l;
    }
}

template <int TYPE, int D>
int launch(const PagedArgs& A, bool split, unsigned grid, cudaStream_t st) {
    constexpr int smem = Shape<TYPE, D>::SMEM;
    static unsigned long long devs_set = 0;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return -1;
    const unsigned long long bit = 1ull << (dev & 63);
    if (!(__atomic_load_n(&devs_set, __ATOMIC_ACQUIRE) & bit)) {
        if (cudaFuncSetAttribute(k_paged<TYPE, D, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess ||
            cudaFuncSetAttribute(k_paged<TYPE, D, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
            return -1;
        __atomic_fetch_or(&devs_set, bit, __ATOMIC_RELEASE);
    }
    if (!split) return kx::launch_pdl(k_paged<TYPE, D, false>, dim3(grid), dim3(PG_THREADS), smem, st, A);
    if (kx::launch_pdl(k_paged<TYPE, D, true>, dim3(grid), dim3(PG_THREADS), smem, st, A) != 0) return -1;
    return kx::launch_pdl(k_paged_join, dim3(grid - 1, A.per_chunk), dim3(128), 0, st, A);
}

template <int TYPE>
int launch_d(const PagedArgs& A, bool split, unsigned grid, cudaStream_t st) {
    return A.c.dk <= 64 && A.c.dv <= 64 ? launch<TYPE, 64>(A, split, grid, st) : launch<TYPE, 128>(A, split, grid, st);
}

}  // namespace

extern "C" {

size_t kx_attention_paged_ws(const kx_kv* c, int H, int n) {
    if (!kx::kv_ok(c) || c->dk > PG_DMAX || c->dv > PG_DMAX || H < 1 || H % c->heads || n < 0) return 0;
    return part_offset(PG_MAX_CTAS, 0);
}

int kx_attention_paged(const kx_kv* c, int layer, const float* q, int ldq, int H, const int32_t* seqs, int n, int window, int sinks,
                       float scale, float* ctx, int ldc, void* ws, size_t ws_bytes, int* status, void* stream) {
    const size_t need = kx_attention_paged_ws(c, H, n);
    if (need == 0 || layer < 0 || layer >= c->layers || sinks < 0 || !std::isfinite(scale)) return -1;
    if (!seqs && n > c->n_seqs) return -1;
    if (n == 0) return 0;
    if (!q || !ctx || ldq < static_cast<long>(H) * c->dk || ldc < static_cast<long>(H) * c->dv) return -1;
    if (!ws || (reinterpret_cast<uintptr_t>(ws) & 15) || ws_bytes < need) return -1;
    const long sz = kx::kv_elem_bytes(c->type);
    PagedArgs A;
    A.c = *c;
    A.k = static_cast<const char*>(c->k) + (layer ? layer * c->k_layer * sz : 0);
    A.v = static_cast<const char*>(c->v) + (layer ? layer * c->v_layer * sz : 0);
    A.q = q;
    A.ctx = ctx;
    A.seqs = seqs;
    A.ws = static_cast<char*>(ws);
    A.status = status;
    A.n = n;
    A.H = H;
    A.G = H / c->heads;
    A.chunks = (A.G + PG_HEADS - 1) / PG_HEADS;
    A.per_chunk = (A.G + A.chunks - 1) / A.chunks;
    A.chunks = (A.G + A.per_chunk - 1) / A.per_chunk;
    A.ldq = ldq;
    A.ldc = ldc;
    A.window = window;
    A.sinks = sinks;
    A.scale2 = (scale == 0.0f ? 1.0f / sqrtf(static_cast<float>(c->dk)) : scale) * 1.4426950408889634f;
    A.vecq = (ldq & 3) == 0 && (c->dk & 3) == 0 && (reinterpret_cast<uintptr_t>(q) & 15) == 0;
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0)
        return -1;
    const long units = static_cast<long>(n) * c->heads * A.chunks;
    if (units > INT32_MAX) return -1;
    // the most steps a head can have: where a range's least length covers them, a CTA per head needs no join
    const int ks = c->type == KX_KV_F32 ? 8 : 16;
    long keys = static_cast<long>(c->max_pages) * c->page;
    if (window > 0) keys = std::min(keys, static_cast<long>(window) + sinks + 2 * ks);
    const bool split = (keys + ks - 1) / ks > PG_MIN_STEPS;
    A.grid = std::min(2 * sms, PG_MAX_CTAS);
    const unsigned grid = split ? A.grid : static_cast<unsigned>(units);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (c->type == KX_KV_F32) return launch_d<KX_KV_F32>(A, split, grid, st);
    if (c->type == KX_KV_F16) return launch_d<KX_KV_F16>(A, split, grid, st);
    return launch_d<KX_KV_BF16>(A, split, grid, st);
}

}  // extern "C"
