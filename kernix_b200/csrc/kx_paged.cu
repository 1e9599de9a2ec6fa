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
//       f16:  2 parts of 11 bits, q scaled by a power of two per head to use f16's range, p in [0, 2^13] relative to the
//             head's largest score in the step;
//       bf16: 3 parts of 8 bits, the third as a second product, or in rows 4-7 where the tile has at most four heads
//             (half the matrix instructions: 32 ragged rows 20.2 -> 18.2 us of GPU time);
//       f32:  tf32 halves, q.k = qh.kh + ql.kh + qh.kl (and p.v likewise), 11 + 11 bits.
//     That keeps fp32's accuracy (parts lost: below 2^-22 of the operand). A step's p.v is added to the output in
//     fp32 registers by CUDA-core adds, not carried through the tensor core's truncating accumulation.
//   * Loads: a warp copies (cp.async) its steps' rows into a ring of its own in shared memory: deep prefetch without
//     registers and without barriers between warps. The order of the reduction axis inside a product is free, so 16
//     contiguous bytes serve a lane as matrix fragments as they lie; masked keys are zero-filled and never read.
//   * Work split: the steps of all rows and heads form one line, cut into equal ranges, one per warp (eight warps per
//     SM); a range may cover several short sequences or a part of a long one. A head whose steps lie in several ranges
//     is joined by a second launch (programmatic dependent) in the order of the ranges: nothing depends on timing.
//     (One range per CTA, its warps meeting in shared memory at every unit, took 80 us for 32 ragged rows of which many
//     are short, this takes 23: the CTA that got the short ones paid the meeting for each.)
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "kx_act.cuh"
#include "kx_kernels.h"
#include "kx_kv.cuh"
#include "kx_pdl.cuh"
#include "kx_sm100.cuh"

namespace {

constexpr unsigned FULL = 0xFFFFFFFFu;
constexpr int PG_WARPS = 4, PG_THREADS = PG_WARPS * 32;
constexpr int PG_STAGES = 3;
constexpr int PG_CTAS = 2;        // per SM (three, with registers for each, measured up to 10 % slower)
constexpr int PG_HEADS = 8;       // query heads per tile
constexpr int PG_MAX_WARPS = 1280;  // of a launch over the line: sizes the workspace
// a warp's range is at least this long: one row of 640 keys took 9.7 us with 2, 12.5 with 4, 15.8 with 8
constexpr int PG_MIN_STEPS = 2;
// a unit's place on the line before its steps: its q, its output (32 ragged bf16 rows: 26.7 us with 1, 24.7 with 3,
// 27.7 with 6)
constexpr int PG_UNIT_COST = 3;
// Units of few steps at most get a CTA each, which joins its warps itself: 5.8 us for 12 steps of 4 units where the line
// and its join take 11. Whether lengths are near their bound is not known here, so the bound grows with the units: 40 steps
// of 64 units 13.1 us against 14.2, of 4 units 12.2 against 9.7; 80 steps of 800 units 84 us against 97, of 64 units 22
// against 19.
inline bool pg_by_units(long steps, long units, int sms) {
    return steps <= 32 || (steps <= 48 && units >= 64) || (steps <= 96 && units >= 4l * sms);
}
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
    int ldq, ldc, window, sinks;
    float scale2;
    bool vecq, vecc;
};

// what a warp's range begins with: written by the main launch, read by the join
struct PagedDesc {
    long long first;  // position of the unit's first step on the line
    long long per;    // length of a range
    int row, unit, last, pad;  // last: the warp whose range the unit ends in
};

// the steps of a row's token: the steps that hold its first tokens, then those of its window
struct Span {
    int len, s0, w0;    // visible: j < s0 or w0 <= j < len
    int na, b0, steps;  // steps 0 .. na - 1, then b0, b0 + 1, ...
    bool bad;           // the row's slot or length is out of range
};
template <int KS>
__device__ __forceinline__ int steps_of(int keys) { return static_cast<int>((static_cast<unsigned>(keys) + KS - 1) / KS); }
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
    sp.na = steps_of<KS>(sp.s0);
    sp.b0 = max(sp.na, sp.w0 / KS);
    sp.steps = max(1, sp.na + steps_of<KS>(len) - sp.b0);  // a row that sees nothing still has its zeros to write
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
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(d[0]), "f"(d[1]), "f"(d[2]), "f"(d[3]));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(d[0]), "f"(d[1]), "f"(d[2]), "f"(d[3]));
}
__device__ __forceinline__ void mma_tf32(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(d[0]), "f"(d[1]), "f"(d[2]), "f"(d[3]));
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
// v = hi + rest with 11 bits in hi, to nearest: rest is at most 2^-12 of v and the tensor core cuts it to 11 bits, 2^-22
// of v at most (cutting hi off as well saves an instruction and costs four times the error). |v| < 2^127.
__device__ __forceinline__ uint32_t tf32_of(float v, float* rest) {
    const uint32_t hi = (__float_as_uint(v) + 0x1000u) & 0xFFFFE000u;
    *rest = v - __uint_as_float(hi);
    return hi;
}

// FEW: a bf16 cache and at most four heads per tile, whose rows 4-7 then take the third parts
template <int TYPE, int D, bool FEW = false>
struct Shape {
    static constexpr int EPC = TYPE == KX_KV_F32 ? 4 : 8;   // elements per 16-byte chunk
    static constexpr int KT = TYPE == KX_KV_F32 ? 1 : 2;    // tiles of 8 keys per step
    static constexpr int KS = 8 * KT;                       // keys per step
    static constexpr int CPR = D / EPC;                     // chunks per row
    static constexpr int PITCH = (CPR + 7) / 8 * 128;       // bytes from row to row in shared memory
    static constexpr int KCH = CPR / 4;                     // K chunks per lane and tile: chunk 4 c + t
    static constexpr int VK = 2 * KT;                       // V keys per lane
    static constexpr int VCH = (CPR + 7) / 8;               // V chunks per lane and key
    static constexpr int NO = VCH * 2 * EPC;                // output elements per lane
    static constexpr int DV = VCH * 8 * EPC;                // a head's outputs, the padding included
    static constexpr int TILE = KS * PITCH;                 // K or V of a step
    static constexpr int STAGE = 2 * TILE;                  // bytes per warp and stage
    static constexpr int QW = D / 4;                        // q elements per lane
    static constexpr int PARTS = TYPE == KX_KV_BF16 ? 3 : 2;
    static constexpr int KEPT = FEW ? 2 : PARTS;                // parts in a lane's registers
    static constexpr int QP = TYPE == KX_KV_F32 ? QW : QW / 2;  // 32-bit words per part
    static constexpr int SMEM = PG_WARPS * PG_STAGES * STAGE;
    static_assert(PG_STAGES * STAGE >= PG_HEADS * DV * 4, "a warp's ring holds its partial output");
};

// where a warp is on the line: step i of unit `unit` (key-value head x tile of heads) of row `row`
template <int TYPE, int D>
struct Cursor {
    using S = Shape<TYPE, D>;
    Span sp;
    int row, slot, unit, i;
    long long pos;  // on the line

    __device__ __forceinline__ void seek_row(const PagedArgs& A, int r) {  // rows that are left alone have no steps
        do {
            row = r++;
            sp = span_of<S::KS>(A, row, &slot);
        } while (sp.steps == 0);
    }
    // to the first step of the next unit, or of none if that lies at `end` or behind it
    __device__ __forceinline__ bool next_unit(const PagedArgs& A, int units, long long end) {
        pos += sp.steps - i + PG_UNIT_COST;
        if (pos >= end) return false;
        i = 0;
        if (++unit == units) {
            unit = 0;
            seek_row(A, row + 1);
        }
        return true;
    }
    __device__ __forceinline__ int first_key() const { return (i < sp.na ? i : i - sp.na + sp.b0) * S::KS; }
    // every key of the step is seen
    __device__ __forceinline__ bool whole() const {
        const int j = first_key();
        return sp.len - j >= S::KS && (j >= sp.w0 || sp.s0 - j >= S::KS);
    }
    __device__ __forceinline__ bool visible(int j) const { return j < sp.len && (j < sp.s0 || j >= sp.w0); }
};

// The loads of a warp: page ids 32 at a time (one per lane), then every lane the chunks of a step that it will use.
template <int TYPE, int D>
struct Feed {
    using S = Shape<TYPE, D>;
    static constexpr long SZ = 16 / S::EPC;
    const int32_t* table;
    const char *kb, *vb;
    int ids, base;  // ids: table[base + lane]

    __device__ __forceinline__ bool held(int entry) const { return static_cast<unsigned>(entry) - static_cast<unsigned>(base) < 32u; }

    __device__ __forceinline__ void unit(const PagedArgs& A, const Cursor<TYPE, D>& c) {
        const int kvh = c.unit / A.chunks;
        table = A.c.table + static_cast<long>(c.slot < A.c.n_seqs ? c.slot : 0) * A.c.max_pages;
        kb = A.k + static_cast<long>(kvh) * A.c.page * A.c.dk * SZ;
        vb = A.v + static_cast<long>(kvh) * A.c.page * A.c.dv * SZ;
        base = -64;
    }
    // Rows (keys) of PITCH bytes, chunk x of row r at place x ^ (r & 7): eight lanes that read the same chunk of eight
    // rows, or four chunks of rows r and r + 4, meet no bank twice. Eight lanes copy 128 contiguous bytes of a row (lanes
    // that copied just what they use themselves asked for 64 bytes at a time: no barrier, but 4.7 TB/s where this reads
    // at 5.8); lane offsets are the same in every step. Chunks behind a row's end are left as they are (zero_pads); rows
    // that are not seen become zero. false: a page that a visible key lies on is not there; its row is zero, too.
    __device__ __forceinline__ bool issue(const PagedArgs& A, const Cursor<TYPE, D>& c, uint32_t dst, int nck, int ncv, int shift) {
        const int lane = threadIdx.x & 31, first = c.first_key(), lr = lane >> 3, lc = lane & 7;
        if (!held(first >> shift) || !held((first + S::KS - 1) >> shift)) {
            base = first >> shift;
            ids = lane <= ((c.sp.len - 1) >> shift) - base ? __ldcg(table + base + lane) : 0;
        }
        // rows lr + 4 y, chunks lc + 8 x
        const uint32_t to[2] = {dst + lr * S::PITCH + ((lc ^ lr) << 4), dst + lr * S::PITCH + ((lc ^ lr ^ 4) << 4)};
        const int p0 = __shfl_sync(FULL, ids, (first >> shift) - base);
        if (A.c.page >= S::KS && c.whole() && p0 >= 0 && p0 < A.c.n_pages) {  // one page, every key seen
            const int slot = (first & (A.c.page - 1)) + lr;
            const char* ks = kb + p0 * A.c.k_page * SZ + (static_cast<long>(slot) * nck + lc) * 16;
            const char* vs = vb + p0 * A.c.v_page * SZ + (static_cast<long>(slot) * ncv + lc) * 16;
#pragma unroll
            for (int y = 0; y < S::KS / 4; y++, ks += 64 * nck)
#pragma unroll
                for (int x = 0; x < S::VCH; x++)
                    if (lc + 8 * x < nck) cp16(to[y & 1] + y * 4 * S::PITCH + x * 128, ks + x * 128, true);
#pragma unroll
            for (int y = 0; y < S::KS / 4; y++, vs += 64 * ncv)
#pragma unroll
                for (int x = 0; x < S::VCH; x++)
                    if (lc + 8 * x < ncv) cp16(to[y & 1] + S::TILE + y * 4 * S::PITCH + x * 128, vs + x * 128, true);
            return true;
        }
        bool good = true;
#pragma unroll
        for (int y = 0; y < S::KS / 4; y++) {
            const int j = first + lr + 4 * y, p = __shfl_sync(FULL, ids, (j >> shift) - base);
            const bool see = c.visible(j), ok = see && p >= 0 && p < A.c.n_pages;
            good = good && (ok || !see);
            const long slot = j & (A.c.page - 1);
            const char* ks = ok ? kb + p * A.c.k_page * SZ + (slot * nck + lc) * 16 : A.k;
            const char* vs = ok ? vb + p * A.c.v_page * SZ + (slot * ncv + lc) * 16 : A.v;
#pragma unroll
            for (int x = 0; x < S::VCH; x++) {
                if (lc + 8 * x < nck) cp16(to[y & 1] + y * 4 * S::PITCH + x * 128, ok ? ks + x * 128 : A.k, ok);
                if (lc + 8 * x < ncv) cp16(to[y & 1] + S::TILE + y * 4 * S::PITCH + x * 128, ok ? vs + x * 128 : A.v, ok);
            }
        }
        return good;
    }
    // the chunks behind dk, which no copy writes, count in the scores as zeros
    __device__ __forceinline__ static void zero_pads(uint8_t* rows, int nck) {
        if (nck == S::CPR) return;
        for (int x = (threadIdx.x & 31) * 16; x < PG_STAGES * S::STAGE; x += 512) *reinterpret_cast<uint4*>(rows + x) = make_uint4(0, 0, 0, 0);
        __syncwarp();
    }
};

// One tile of query heads against the cache: q's parts, and the running maximum (in base 2), sum and output. Lane
// (g, t) holds head g; after the last step its sum is that of its own columns only.
// Column n of a tile's scores is the key in row (n >> 1) + 4 (n & 1) of its eight (a lane's columns 2 t and 2 t + 1:
// rows t and t + 4), and lane g reads its values in chunk (g >> 1) + 4 (g & 1) of eight: the orders without conflicts.
template <int TYPE, int D, bool FEW>
struct Tile {
    using S = Shape<TYPE, D, FEW>;
    uint32_t qp[S::KEPT][S::QP];
    float2 o[S::NO / 2];  // o[EPC c + e]: elements e of chunks 8 c + t and 8 c + t + 4
    float m, l, qscale, off;

    // x: the head's q, lane t the elements that its K chunks hold
    __device__ __forceinline__ void start(const PagedArgs& A, const Cursor<TYPE, D>& c) {
        const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
        const int kvh = c.unit / A.chunks, head0 = kvh * A.G + (c.unit - kvh * A.chunks) * A.per_chunk;
        const int heads = min(A.per_chunk, (kvh + 1) * A.G - head0);
        const float* qr = A.q + static_cast<long>(c.row) * A.ldq + static_cast<long>(head0 + min(FEW ? g & 3 : g, heads - 1)) * A.c.dk;
        float x[S::QW];
#pragma unroll
        for (int k = 0; k < S::KCH; k++)
#pragma unroll
            for (int e = 0; e < S::EPC; e += 4) {
                const int d = (k * 4 + t) * S::EPC + e;
                float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
                if (d < A.c.dk) f = A.vecq ? *reinterpret_cast<const float4*>(qr + d) : make_float4(qr[d], qr[d + 1], qr[d + 2], qr[d + 3]);
                x[k * S::EPC + e] = f.x;
                x[k * S::EPC + e + 1] = f.y;
                x[k * S::EPC + e + 2] = f.z;
                x[k * S::EPC + e + 3] = f.w;
            }
        qscale = A.scale2;
        // weights up to 2^off: below 1 / len, so that no sum of weighted values passes the largest value
        off = static_cast<float>(__clz(c.sp.len) - 32);
        if constexpr (TYPE == KX_KV_F16) {
            // |q| < 2^14 after the scaling; parts keep 22 bits of what is above 2^-17 of the head's largest element
            float top = 0.0f;
#pragma unroll
            for (int k = 0; k < S::QW; k++) top = fmaxf(top, fabsf(x[k]));
            top = fmaxf(top, __shfl_xor_sync(FULL, top, 1));
            top = fmaxf(top, __shfl_xor_sync(FULL, top, 2));
            const int e = min(max(static_cast<int>(__float_as_uint(top) >> 23) - 127, -100), 126);  // floor(log2 top)
            const float up = __uint_as_float(static_cast<uint32_t>(127 + 13 - e) << 23);
            qscale *= __uint_as_float(static_cast<uint32_t>(127 - 13 + e) << 23);
            off = 13.0f;
#pragma unroll
            for (int k = 0; k < S::QW; k++) x[k] *= up;
        }
        if constexpr (TYPE == KX_KV_F32) {
#pragma unroll
            for (int k = 0; k < S::QW; k++) {
                float lo;
                qp[0][k] = tf32_of(x[k], &lo);
                qp[1][k] = __float_as_uint(lo);
            }
        } else {
#pragma unroll
            for (int k = 0; k < S::QP; k++) {
                float a = x[2 * k], b = x[2 * k + 1];
                uint32_t w[S::PARTS];
#pragma unroll
                for (int p = 0; p < S::PARTS; p++) w[p] = pack2<TYPE>(a, b, &a, &b);
#pragma unroll
                for (int p = 0; p < S::KEPT; p++) qp[p][k] = w[p];
                if (FEW && g >= 4) qp[0][k] = w[S::PARTS - 1], qp[1][k] = 0;
            }
        }
#pragma unroll
        for (int k = 0; k < S::NO / 2; k++) o[k] = make_float2(0.0f, 0.0f);
        m = -INFINITY;
        l = 0.0f;
    }

    // a step whose rows lie at src in shared memory
    __device__ __forceinline__ void step(const Cursor<TYPE, D>& c, const uint8_t* src) {
        const int g = threadIdx.x >> 2 & 7, t = threadIdx.x & 3, perm = (g >> 1) | (g & 1) << 2;
        const uint8_t* krow = src + perm * S::PITCH;
        const int kch[2] = {(t ^ (perm & 3) | (perm & 4)) << 4, (t ^ (perm & 3) | (~perm & 4)) << 4};
        // scores: rows 0-7 and 8-15 of the tile are the products of q's parts
        float s[2 * S::KT];
#pragma unroll
        for (int u = 0; u < S::KT; u++) {
            float dd[4][4] = {};  // chains of products: by even and odd chunk, and the last part's apart
#pragma unroll
            for (int k = 0; k < S::KCH; k++) {
                float(&d)[4] = dd[k & 1];
                float(&f)[4] = dd[2 + (k & 1)];
                const uint4 kv = *reinterpret_cast<const uint4*>(krow + u * 8 * S::PITCH + (k >> 1) * 128 + kch[k & 1]);
                const int x = k * 4;
                if constexpr (TYPE == KX_KV_F32) {
                    const uint32_t w[4] = {kv.x, kv.y, kv.z, kv.w};
#pragma unroll
                    for (int h = 0; h < 4; h += 2) {
                        float l0, l1;
                        const uint32_t h0 = tf32_of(__uint_as_float(w[h]), &l0), h1 = tf32_of(__uint_as_float(w[h + 1]), &l1);
                        mma_tf32(d, qp[0][x + h], qp[1][x + h], qp[0][x + h + 1], qp[1][x + h + 1], h0, h1);
                        mma_tf32(f, qp[0][x + h], 0, qp[0][x + h + 1], 0, __float_as_uint(l0), __float_as_uint(l1));
                    }
                } else if constexpr (TYPE == KX_KV_F16) {
                    mma_f16(d, qp[0][x], qp[1][x], qp[0][x + 1], qp[1][x + 1], kv.x, kv.y);
                    mma_f16(d, qp[0][x + 2], qp[1][x + 2], qp[0][x + 3], qp[1][x + 3], kv.z, kv.w);
                } else {
                    mma_bf16(d, qp[0][x], qp[1][x], qp[0][x + 1], qp[1][x + 1], kv.x, kv.y);
                    mma_bf16(d, qp[0][x + 2], qp[1][x + 2], qp[0][x + 3], qp[1][x + 3], kv.z, kv.w);
                    if constexpr (!FEW) {
                        mma_bf16(f, qp[2][x], 0, qp[2][x + 1], 0, kv.x, kv.y);
                        mma_bf16(f, qp[2][x + 2], 0, qp[2][x + 3], 0, kv.z, kv.w);
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < 2; e++)
                // rounded here for good: a product that reached the exponential unrounded would pass its own maximum
                s[2 * u + e] = __fmul_rn((dd[0][e] + dd[1][e]) + ((dd[0][e + 2] + dd[1][e + 2]) + (dd[2][e] + dd[3][e])), qscale);
            if (FEW) {
#pragma unroll
                for (int e = 0; e < 2; e++) s[2 * u + e] += __shfl_xor_sync(FULL, s[2 * u + e], 16);
            }
        }
        if (!c.whole()) {
            const int j = c.first_key() + t;
#pragma unroll
            for (int e = 0; e < 2 * S::KT; e++)
                if (!c.visible(j + e * 4)) s[e] = -INFINITY;
        }
        float mx = s[0];
#pragma unroll
        for (int e = 1; e < 2 * S::KT; e++) mx = fmaxf(mx, s[e]);
        mx = fmaxf(mx, __shfl_xor_sync(FULL, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(FULL, mx, 2));
        const float mn = fmaxf(m, mx);
        const float safe = mn == -INFINITY ? 0.0f : mn;
        if (__any_sync(FULL, mn > m)) {
            const float alpha = kx::ex2_approx(m - safe);
            l *= alpha;
#pragma unroll
            for (int e = 0; e < S::NO / 2; e++) o[e].x *= alpha, o[e].y *= alpha;
        }
        m = mn;
        // Weights as f16 parts keep 2^-38 of what they are relative to: that is the head's largest score in the step, not
        // its running maximum, so that a step of small weights and large values keeps its bits; its products join the
        // output by the step's share.
        constexpr bool LOCAL = TYPE == KX_KV_F16;
        const float peak = LOCAL ? (mx == -INFINITY ? 0.0f : mx) : safe, share = LOCAL ? kx::ex2_approx(mx - safe) : 1.0f;
        float p[2 * S::KT], sum = LOCAL ? 0.0f : l;
#pragma unroll
        for (int e = 0; e < 2 * S::KT; e++) {
            p[e] = kx::ex2_approx((s[e] - peak) + off);  // the largest is 2^off, however large the scores are
            sum += p[e];
        }
        l = LOCAL ? fmaf(sum, share, l) : sum;
        // p.v: column 2 t (2 t + 1) of n-tile (k, e) is element e of chunk 8 k + t (+ 4); row t + 4 x of the step is x-th
        const uint8_t* vrow = src + S::TILE + t * S::PITCH;
        const int vch[2] = {(perm ^ t) << 4, (perm ^ t ^ 4) << 4};
        const auto values = [&](int x, int k) { return *reinterpret_cast<const uint4*>(vrow + x * 4 * S::PITCH + k * 128 + vch[x & 1]); };
        if constexpr (TYPE == KX_KV_F32) {
            float q0, q1;
            const uint32_t h0 = tf32_of(p[0], &q0), h1 = tf32_of(p[1], &q1);
#pragma unroll
            for (int k = 0; k < S::VCH; k++) {
                const uint4 va = values(0, k), vb = values(1, k);
                const uint32_t wa[4] = {va.x, va.y, va.z, va.w}, wb[4] = {vb.x, vb.y, vb.z, vb.w};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float d[4] = {0.f, 0.f, 0.f, 0.f}, l0, l1;
                    const uint32_t v0 = tf32_of(__uint_as_float(wa[e]), &l0), v1 = tf32_of(__uint_as_float(wb[e]), &l1);
                    mma_tf32(d, h0, 0, h1, 0, __float_as_uint(l0), __float_as_uint(l1));
                    mma_tf32(d, h0, __float_as_uint(q0), h1, __float_as_uint(q1), v0, v1);
                    o[k * 4 + e] = kx::add2(o[k * 4 + e], kx::add2(make_float2(d[0], d[1]), make_float2(d[2], d[3])));
                }
            }
        } else {
            uint32_t pa[S::PARTS], pb[S::PARTS];
            {
                float a = p[0], b = p[1], cc = p[2], d = p[3];
#pragma unroll
                for (int x = 0; x < S::PARTS; x++) {
                    pa[x] = pack2<TYPE>(a, b, &a, &b);
                    pb[x] = pack2<TYPE>(cc, d, &cc, &d);
                }
                if (FEW && g >= 4) pa[0] = pa[S::PARTS - 1], pb[0] = pb[S::PARTS - 1], pa[1] = pb[1] = 0;
            }
#pragma unroll
            for (int k = 0; k < S::VCH; k++) {
                uint32_t w[4][4];
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const uint4 x = values(u, k);
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
                        if constexpr (!FEW) mma_bf16(d, pa[2], 0, pb[2], 0, b0, b1);
                        mma_bf16(d, pa[0], pa[1], pb[0], pb[1], b0, b1);
                    }
                    const float2 pv = kx::add2(make_float2(d[0], d[1]), make_float2(d[2], d[3]));
                    o[k * 8 + e] = LOCAL ? kx::fma2(pv, make_float2(share, share), o[k * 8 + e]) : kx::add2(o[k * 8 + e], pv);
                }
            }
        }
    }

    __device__ __forceinline__ void finish(bool bad) {
        l += __shfl_xor_sync(FULL, l, 1);
        l += __shfl_xor_sync(FULL, l, 2);
        if (bad) l = NAN;
        if (FEW) {
#pragma unroll
            for (int k = 0; k < S::NO / 2; k++) {
                o[k].x += __shfl_xor_sync(FULL, o[k].x, 16);
                o[k].y += __shfl_xor_sync(FULL, o[k].y, 16);
            }
        }
    }
    // outputs e .. e + 3 of chunk group k: element d of the head
    __device__ __forceinline__ static int element(int k, int e) {
        return (k * 8 + (threadIdx.x & 3)) * S::EPC + (e < S::EPC ? e : e + 3 * S::EPC);
    }
    __device__ __forceinline__ float4 four(int k, int e, float f) const {
        const float2* x = o + k * S::EPC + e % S::EPC;
        return e < S::EPC ? make_float4(x[0].x * f, x[1].x * f, x[2].x * f, x[3].x * f)
                          : make_float4(x[0].y * f, x[1].y * f, x[2].y * f, x[3].y * f);
    }
};

constexpr size_t PG_PART = (PG_HEADS * PG_DMAX + 2 * PG_HEADS) * sizeof(float);
__device__ __host__ inline size_t part_offset(int warp, int which) {
    return PG_MAX_WARPS * sizeof(PagedDesc) + (static_cast<size_t>(warp) * 2 + which) * PG_PART;
}

__device__ __forceinline__ int tile_heads(const PagedArgs& A, int unit, int* head0) {
    const int kvh = unit / A.chunks;
    *head0 = kvh * A.G + (unit - kvh * A.chunks) * A.per_chunk;
    return min(A.per_chunk, (kvh + 1) * A.G - *head0);
}

// Short sequences: one CTA per unit, its warps take every fourth step and meet in shared memory.
template <int TYPE, int D, bool FEW>
__global__ void __launch_bounds__(PG_THREADS, PG_CTAS) k_paged_unit(const PagedArgs A) {
    using S = Shape<TYPE, D>;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float red[PG_WARPS][PG_HEADS][2];
    const int units = A.c.heads * A.chunks, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int nck = A.c.dk / S::EPC, ncv = A.c.dv / S::EPC, shift = 31 - __clz(A.c.page);
    kx::griddep_wait();
    kx::griddep_launch_dependents();
    Cursor<TYPE, D> c;
    c.row = blockIdx.x / units;
    c.unit = blockIdx.x - c.row * units;
    c.sp = span_of<S::KS>(A, c.row, &c.slot);
    if (c.sp.steps == 0) return;
    uint8_t* const rows = smem + warp * (PG_STAGES * S::STAGE);
    const uint32_t ring = kx::smem_u32(rows);
    Feed<TYPE, D>::zero_pads(rows, nck);
    Feed<TYPE, D> feed;
    feed.unit(A, c);
    bool bad = c.sp.bad;
    Cursor<TYPE, D> ahead = c;
    ahead.i = warp;
    const auto issue = [&](int stage) {
        if (ahead.i < c.sp.steps && !feed.issue(A, ahead, ring + stage * S::STAGE, nck, ncv, shift)) bad = true;
        ahead.i += PG_WARPS;
        cp_commit();
    };
#pragma unroll
    for (int s = 0; s < PG_STAGES - 1; s++) issue(s);
    Tile<TYPE, D, FEW> tile;
    tile.start(A, c);
    int stage = 0;
    for (c.i = warp; c.i < c.sp.steps; c.i += PG_WARPS) {
        __syncwarp();  // every lane has read the rows of the step before
        issue(stage == 0 ? PG_STAGES - 1 : stage - 1);
        cp_wait<PG_STAGES - 1>();
        __syncwarp();  // every lane's copies of this step are there
        tile.step(c, rows + stage * S::STAGE);
        stage = stage + 1 == PG_STAGES ? 0 : stage + 1;
    }
    cp_wait<0>();
    bad = __any_sync(FULL, bad);
    if (bad && lane == 0) kx::kv_report(A.status, KX_STATUS_BAD_REQUEST);
    tile.finish(bad);
    if (t == 0) {
        red[warp][g][0] = tile.m;
        red[warp][g][1] = tile.l;
    }
    __syncwarp();
    float* mine = reinterpret_cast<float*>(smem + warp * (PG_STAGES * S::STAGE));  // the warp's ring, no longer in use
#pragma unroll
    for (int k = 0; k < S::VCH; k++)
#pragma unroll
        for (int e = 0; e < 2 * S::EPC; e += 4) *reinterpret_cast<float4*>(mine + g * S::DV + tile.element(k, e)) = tile.four(k, e, 1.0f);
    __syncthreads();
    int head0;
    const int heads = tile_heads(A, c.unit, &head0);
    for (int x = tid; x < heads * S::DV; x += PG_THREADS) {
        const int h = x / S::DV, d = x - h * S::DV;
        float mm = red[0][h][0];
#pragma unroll
        for (int w = 1; w < PG_WARPS; w++) mm = fmaxf(mm, red[w][h][0]);
        const float ms = mm == -INFINITY ? 0.0f : mm;
        float num = 0.0f, den = 0.0f;
#pragma unroll
        for (int w = 0; w < PG_WARPS; w++) {
            const float f = kx::ex2_approx(red[w][h][0] - ms);
            den += f * red[w][h][1];
            num += f * reinterpret_cast<const float*>(smem + w * (PG_STAGES * S::STAGE))[x];
        }
        if (d < A.c.dv) A.ctx[static_cast<long>(c.row) * A.ldc + static_cast<long>(head0 + h) * A.c.dv + d] = den == 0.0f ? 0.0f : num / den;
    }
}

// Warp w of the launch takes the steps [w per, (w + 1) per) of the line, whatever units they belong to; the loads run
// ahead of the products across the units' ends.
template <int TYPE, int D, bool FEW>
__global__ void __launch_bounds__(PG_THREADS, PG_CTAS) k_paged_line(const PagedArgs A) {
    using S = Shape<TYPE, D>;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ long long upto[PG_THREADS];
    __shared__ long long sums[PG_WARPS];
    const int units = A.c.heads * A.chunks, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int nck = A.c.dk / S::EPC, ncv = A.c.dv / S::EPC, shift = 31 - __clz(A.c.page);
    kx::griddep_wait();
    kx::griddep_launch_dependents();

    // rows r0 .. r0 + PG_THREADS - 1: upto[x] = a unit's length on the line, summed over the rows r0 .. r0 + x; returns
    // the last of them
    const auto scan_rows = [&](int r0) {
        int slot;
        const int r = r0 + tid;
        long long v = r < A.n ? span_of<S::KS>(A, r, &slot).steps : 0;
        if (v > 0) v += PG_UNIT_COST;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const long long u = __shfl_up_sync(FULL, v, d);
            if (lane >= d) v += u;
        }
        __syncthreads();
        if (lane == 31) sums[warp] = v;
        __syncthreads();
        long long all = 0;
#pragma unroll
        for (int w = 0; w < PG_WARPS; w++) {
            if (w < warp) v += sums[w];
            all += sums[w];
        }
        upto[tid] = v;
        __syncthreads();
        return all;
    };
    long long total = 0;
    for (int r0 = 0; r0 < A.n; r0 += PG_THREADS) total += scan_rows(r0);
    total *= units;
    const int me = blockIdx.x * PG_WARPS + warp, warps = gridDim.x * PG_WARPS;
    const long long per = max((total + warps - 1) / warps, static_cast<long long>(PG_MIN_STEPS));
    const long long lo = me * per, hi = min(lo + per, total);
    Cursor<TYPE, D> c;
    c.row = -1;
    long long first = 0;  // where the row begins
    long long before = 0;
    for (int r0 = 0; r0 < A.n; r0 += PG_THREADS) {  // the row that lo lies in
        const long long all = A.n > PG_THREADS ? scan_rows(r0) : total / units;
        if (c.row < 0 && lo < total && lo < (before + all) * units) {
#pragma unroll
            for (int x = 0; x < PG_THREADS; x += 32) {
                const unsigned hit = __ballot_sync(FULL, lo < (before + upto[x + lane]) * units);
                if (hit) {
                    const int at = x + __ffs(hit) - 1;
                    c.row = r0 + at;
                    first = (before + (at ? upto[at - 1] : 0)) * units;
                    break;
                }
            }
        }
        before += all;
    }
    PagedDesc* desc = reinterpret_cast<PagedDesc*>(A.ws) + me;
    if (c.row >= 0) {
        c.sp = span_of<S::KS>(A, c.row, &c.slot);
        const int length = c.sp.steps + PG_UNIT_COST;
        c.unit = static_cast<int>((lo - first) / length);
        first += static_cast<long long>(c.unit) * length + PG_UNIT_COST;  // the unit's first step
        c.pos = max(lo, first);
        c.i = static_cast<int>(c.pos - first);
    }
    if (c.row < 0 || c.pos >= hi) {
        if (lane == 0) desc->row = -1;
        return;
    }
    if (lane == 0) *desc = PagedDesc{first, per, c.row, c.unit, static_cast<int>((first + c.sp.steps - 1) / per), 0};

    uint8_t* const rows = smem + warp * (PG_STAGES * S::STAGE);
    const uint32_t ring = kx::smem_u32(rows);
    Feed<TYPE, D>::zero_pads(rows, nck);
    Cursor<TYPE, D> ahead = c;
    Feed<TYPE, D> feed;
    feed.unit(A, ahead);
    unsigned missing = 0;  // per stage: a page was not there
    const auto issue = [&](int stage) {
        if (ahead.pos < hi) {
            const bool good = feed.issue(A, ahead, ring + stage * S::STAGE, nck, ncv, shift);
            missing = (missing & ~(1u << stage)) | (good ? 0u : 1u << stage);
            if (ahead.i + 1 < ahead.sp.steps) {
                ahead.i++;
                ahead.pos++;
            } else if (ahead.next_unit(A, units, hi)) {
                feed.unit(A, ahead);
            }
        }
        cp_commit();
    };
#pragma unroll
    for (int s = 0; s < PG_STAGES - 1; s++) issue(s);
    Tile<TYPE, D, FEW> tile;
    int stage = 0;
    do {
        const int i0 = c.i, steps = static_cast<int>(min(static_cast<long long>(c.sp.steps - c.i), hi - c.pos));
        bool bad = c.sp.bad;
        tile.start(A, c);
        for (int x = 0; x < steps; x++) {
            __syncwarp();  // every lane has read the rows of the step before
            issue(stage == 0 ? PG_STAGES - 1 : stage - 1);
            cp_wait<PG_STAGES - 1>();
            __syncwarp();  // every lane's copies of this step are there
            bad = bad || (missing >> stage & 1);
            c.i = i0 + x;
            tile.step(c, rows + stage * S::STAGE);
            stage = stage + 1 == PG_STAGES ? 0 : stage + 1;
        }
        bad = __any_sync(FULL, bad);
        if (bad && lane == 0) kx::kv_report(A.status, KX_STATUS_BAD_REQUEST);
        tile.finish(bad);
        int head0;
        const int heads = tile_heads(A, c.unit, &head0);
        if (g < heads) {
            if (steps == c.sp.steps) {
                const float inv = tile.l == 0.0f ? 0.0f : 1.0f / tile.l;
                float* out = A.ctx + static_cast<long>(c.row) * A.ldc + static_cast<long>(head0 + g) * A.c.dv;
#pragma unroll
                for (int k = 0; k < S::VCH; k++)
#pragma unroll
                    for (int e = 0; e < 2 * S::EPC; e += 4) {
                        const int d = tile.element(k, e);
                        if (d >= A.c.dv) continue;
                        const float4 f = tile.four(k, e, inv);
                        if (A.vecc) {
                            *reinterpret_cast<float4*>(out + d) = f;
                        } else {
                            out[d] = f.x, out[d + 1] = f.y, out[d + 2] = f.z, out[d + 3] = f.w;
                        }
                    }
            } else {  // a unit in several ranges: its first part in place 1, the others in place 0
                float* part = reinterpret_cast<float*>(A.ws + part_offset(me, i0 == 0));
#pragma unroll
                for (int k = 0; k < S::VCH; k++)
#pragma unroll
                    for (int e = 0; e < 2 * S::EPC; e += 4)
                        *reinterpret_cast<float4*>(part + g * PG_DMAX + tile.element(k, e)) = tile.four(k, e, 1.0f);
                if (t == 0) *reinterpret_cast<float2*>(part + PG_HEADS * PG_DMAX + 2 * g) = make_float2(tile.m, tile.l);
            }
        }
        c.i = i0;
    } while (c.next_unit(A, units, hi));
}

// A unit's parts j .. j1 (warps of the line) for head h, every STRIDE-th from j + begin on: maximum, sum and output (4
// elements per lane), in the parts' order. Eight parts' loads at a time: the loop is a chain of L2 round trips.
template <int STRIDE>
__device__ __forceinline__ void join_parts(const PagedArgs& A, int j, int j1, int h, int begin, float* m, float* den, float4* num) {
    const int d = (threadIdx.x & 31) * 4;
    *m = -INFINITY;
    *den = 0.0f;
    *num = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = j + begin; i <= j1; i += 8 * STRIDE) {
        float4 v[8];
        float2 st[8];
#pragma unroll
        for (int u = 0; u < 8; u++) {
            const int at = i + u * STRIDE;
            const bool in = at <= j1;
            const float* p = reinterpret_cast<const float*>(A.ws + part_offset(in ? at : i, (in ? at : i) == j));
            st[u] = in ? __ldcg(reinterpret_cast<const float2*>(p + PG_HEADS * PG_DMAX + 2 * h)) : make_float2(-INFINITY, 0.0f);
            v[u] = in && d < A.c.dv ? __ldcg(reinterpret_cast<const float4*>(p + h * PG_DMAX + d)) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        float top = *m;
#pragma unroll
        for (int u = 0; u < 8; u++) top = fmaxf(top, st[u].x);
        const float safe = top == -INFINITY ? 0.0f : top, back = kx::ex2_approx(*m - safe);
        *m = top;
        *den *= back;
        num->x *= back, num->y *= back, num->z *= back, num->w *= back;
#pragma unroll
        for (int u = 0; u < 8; u++) {
            const float f = kx::ex2_approx(st[u].x - safe);
            *den += f * st[u].y;
            num->x += f * v[u].x;
            num->y += f * v[u].y;
            num->z += f * v[u].z;
            num->w += f * v[u].w;
        }
    }
}

// Tasks (warp j of the line, head h): if the range of warp j + 1 begins inside a unit whose first step lies in the range
// of warp j, that unit's parts are joined for head h: by one warp where they are few, else by the CTA's eight, each
// every eighth part, then the warps' sums in order.
__global__ void __launch_bounds__(256) k_paged_join(const PagedArgs A, int warps) {
    __shared__ float acc[8][PG_DMAX];
    __shared__ float sum[8], top[8];
    __shared__ int4 todo[2][32];  // few parts, many parts: j, last part, head of the tile, head of the row
    __shared__ int todo_row[2][32], n_todo[2];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    kx::griddep_wait();
    const PagedDesc* desc = reinterpret_cast<const PagedDesc*>(A.ws);
    const int tasks = (warps - 1) * A.per_chunk;
    for (int t0 = blockIdx.x; t0 < tasks; t0 += gridDim.x * 32) {
        if (warp == 0) {
            const int task = t0 + lane * gridDim.x;
            bool hit = false, many = false;
            int4 what = make_int4(0, 0, 0, 0);
            int row = -1;
            if (task < tasks) {
                const int j = task / A.per_chunk, h = task - j * A.per_chunk;
                const longlong2 line = __ldcg(reinterpret_cast<const longlong2*>(&desc[j + 1].first));
                const int4 unit = __ldcg(reinterpret_cast<const int4*>(&desc[j + 1].row));
                if (unit.x >= 0) {
                    int head0;
                    hit = line.x >= j * line.y && line.x < (j + 1) * line.y && h < tile_heads(A, unit.y, &head0);
                    many = unit.z >= j + 16;
                    what = make_int4(j, unit.z, h, head0 + h);
                    row = unit.x;
                }
            }
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const bool mine = hit && many == (x == 1);
                const unsigned hits = __ballot_sync(FULL, mine);
                if (mine) {
                    todo[x][__popc(hits & ((1u << lane) - 1))] = what;
                    todo_row[x][__popc(hits & ((1u << lane) - 1))] = row;
                }
                if (lane == 0) n_todo[x] = __popc(hits);
            }
        }
        __syncthreads();
        float m, den;
        float4 num;
        for (int x = warp; x < n_todo[0]; x += 8) {
            const int4 w = todo[0][x];
            join_parts<1>(A, w.x, w.y, w.z, 0, &m, &den, &num);
            const float inv = den == 0.0f ? 0.0f : 1.0f / den;
            if (lane * 4 < A.c.dv) {
                float* out = A.ctx + static_cast<long>(todo_row[0][x]) * A.ldc + static_cast<long>(w.w) * A.c.dv + lane * 4;
                out[0] = num.x * inv, out[1] = num.y * inv, out[2] = num.z * inv, out[3] = num.w * inv;
            }
        }
        for (int x = 0; x < n_todo[1]; x++) {
            const int4 w = todo[1][x];
            join_parts<8>(A, w.x, w.y, w.z, warp, &m, &den, &num);
            *reinterpret_cast<float4*>(&acc[warp][lane * 4]) = num;
            if (lane == 0) {
                sum[warp] = den;
                top[warp] = m;
            }
            __syncthreads();
            if (tid < A.c.dv) {
                float n = 0.0f, l = 0.0f, all = top[0];
#pragma unroll
                for (int z = 1; z < 8; z++) all = fmaxf(all, top[z]);
                const float safe = all == -INFINITY ? 0.0f : all;
#pragma unroll
                for (int z = 0; z < 8; z++) {
                    const float f = kx::ex2_approx(top[z] - safe);
                    n += f * acc[z][tid];
                    l += f * sum[z];
                }
                A.ctx[static_cast<long>(todo_row[1][x]) * A.ldc + static_cast<long>(w.w) * A.c.dv + tid] = l == 0.0f ? 0.0f : n / l;
            }
            __syncthreads();
        }
        __syncthreads();  // todo is free for the next round
    }
}

template <int TYPE, int D, bool FEW>
int launch(const PagedArgs& A, bool split, unsigned grid, cudaStream_t st) {
    constexpr int smem = Shape<TYPE, D>::SMEM;
    static unsigned long long devs_set = 0;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return -1;
    const unsigned long long bit = 1ull << (dev & 63);
    if (!(__atomic_load_n(&devs_set, __ATOMIC_ACQUIRE) & bit)) {
        if (cudaFuncSetAttribute(k_paged_line<TYPE, D, FEW>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess ||
            cudaFuncSetAttribute(k_paged_unit<TYPE, D, FEW>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
            return -1;
        __atomic_fetch_or(&devs_set, bit, __ATOMIC_RELEASE);
    }
    if (!split) return kx::launch_pdl(k_paged_unit<TYPE, D, FEW>, dim3(grid), dim3(PG_THREADS), smem, st, A);
    if (kx::launch_pdl(k_paged_line<TYPE, D, FEW>, dim3(grid), dim3(PG_THREADS), smem, st, A) != 0) return -1;
    return kx::launch_pdl(k_paged_join, dim3(grid), dim3(256), 0, st, A, static_cast<int>(grid * PG_WARPS));
}

// D: the head dims rounded up to 32; every size runs without a branch inside a step
template <int TYPE, bool FEW>
int launch_d(const PagedArgs& A, bool split, unsigned grid, cudaStream_t st) {
    switch ((std::max(A.c.dk, A.c.dv) + 31) / 32) {
        case 1: return launch<TYPE, 32, FEW>(A, split, grid, st);
        case 2: return launch<TYPE, 64, FEW>(A, split, grid, st);
        case 3: return launch<TYPE, 96, FEW>(A, split, grid, st);
        default: return launch<TYPE, 128, FEW>(A, split, grid, st);
    }
}

}  // namespace

extern "C" {

size_t kx_attention_paged_ws(const kx_kv* c, int H, int n) {
    if (!kx::kv_ok(c) || c->dk > PG_DMAX || c->dv > PG_DMAX || H < 1 || H % c->heads || n < 0) return 0;
    return part_offset(PG_MAX_WARPS, 0);
}

int kx_attention_paged(const kx_kv* c, int layer, const float* q, int ldq, int H, const int32_t* seqs, int n, int window, int sinks,
                       float scale, float* ctx, int ldc, void* ws, size_t ws_bytes, int* status, void* stream) {
    const size_t need = kx_attention_paged_ws(c, H, n);
    if (need == 0 || layer < 0 || layer >= c->layers || sinks < 0 || !std::isfinite(scale * 1.4426950408889634f)) return -1;
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
    A.vecc = (ldc & 3) == 0 && (reinterpret_cast<uintptr_t>(ctx) & 15) == 0;
    A.vecq = (ldq & 3) == 0 && (c->dk & 3) == 0 && (reinterpret_cast<uintptr_t>(q) & 15) == 0;
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0)
        return -1;
    const long units = static_cast<long>(n) * c->heads * A.chunks;
    if (units > INT32_MAX - PG_THREADS) return -1;  // rows are counted in steps of a CTA
    // the most steps a unit can have
    const int ks = c->type == KX_KV_F32 ? 8 : 16;
    long keys = static_cast<long>(c->max_pages) * c->page;
    if (window > 0) keys = std::min(keys, static_cast<long>(window) + sinks + 2 * ks);
    const bool split = !pg_by_units((keys + ks - 1) / ks, units, sms);
    const unsigned grid = split ? std::min(PG_CTAS * sms, PG_MAX_WARPS / PG_WARPS) : static_cast<unsigned>(units);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (c->type == KX_KV_F32) return launch_d<KX_KV_F32, false>(A, split, grid, st);
    if (c->type == KX_KV_F16) return launch_d<KX_KV_F16, false>(A, split, grid, st);
    return A.per_chunk <= 4 ? launch_d<KX_KV_BF16, true>(A, split, grid, st) : launch_d<KX_KV_BF16, false>(A, split, grid, st);
}

}  // extern "C"
