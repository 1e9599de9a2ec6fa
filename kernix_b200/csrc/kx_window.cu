// KERNIX-B200 attention of prompts with a sliding window whose first tokens stay visible (kx_attention_window,
// include/kx_kernels.h), in fp32, on the 5th-generation tensor cores. Per query row at position t and head, over the keys
// j <= t with j > t - window or j < sinks:  ctx = sum_j p_j v_j / sum_j p_j,  p_j = exp(s_j - max s),  s_j = scale q.k_j.
//
// fp32 accuracy from fp16 products: an fp32 value, scaled by a power of two so that the largest of its query row (of its
// 64 keys) is in [2^13, 2^14), is the sum of two fp16 parts up to 2^-22 of itself (up to 2^-39 of that largest where
// that is more), and a.b = ah.bh + al.bh + ah.bl: three fp16 products where 3xTF32 (the same 11-bit parts, no scaling)
// would cost six fp16 products' time. One scale per query row and one per tile of keys and of values: they are undone
// in fp32, the scores' in the exponential's multiply-add, the values' by the factor with which a tile's P.V joins the
// output. p is taken relative to the row's largest score in the tile, not to its running maximum, and becomes p 2^13: it
// keeps 2^-22 of itself, or 2^-38 of that largest where that is more, whatever other tiles hold (relative to the running
// maximum, small weights of a tile of much larger values lost the bits that their products needed).
// (A scale per key and per value column of a tile cost as many instructions as the rest of the softmax together:
// 237 us against 224 for 4096 rows of 16 heads of 128 with a window of 2048, before the steps that made it 179.)
//
//  k_win_prep: per (sample, key-value head, tile of 64 keys) the parts of K (key-major) and V (transposed) in the
//    128-byte-swizzled layout that the matrix instructions read, one contiguous block, so that the main kernel fetches a
//    tile by two bulk copies and every CTA that reads it is spared the conversion. Tiles that no query sees are skipped.
//  k_win_main: one CTA per (sample, key-value head, 128 rows); a row is one query of one of the G heads that share the
//    keys (128 / G queries), so that few queries still fill the tile and a window's edges are short. Two warps fetch K and
//    V tiles (three places each), two issue S = Q.K^T and P.V, and two groups of 128 threads take every second tile:
//    thread = row, S out of tensor memory, maximum, exponentials, P's parts back into tensor memory over S (the A operand
//    of P.V), the tile's P.V added to the row's output in registers. While one group works on its tile the tensor cores
//    work on the other's. Each group keeps a softmax of its own (maximum, sum, output); the two are joined at the end.
//    Sums: S and a tile's P.V are at most 24 accumulated steps in the tensor core, everything longer is fp32 adds.
//    Bound: the chain S -> softmax -> P.V of a group and, close to it, the tensor cores (for heads of 128 a tile's
//    products are 1536 cycles of tensor work; measured 2240 per tile, in which each group's softmax is 1500 of its 4480, before
//    the rounding of large scores and the weights per tile, which cost 1 %)
//    plus a CTA's beginning and end, one fifth of its time. 16384 rows of 16 heads of 128 over 4 key-value heads with a
//    window of 2048: 884 us a call with inputs that change from call to call, 292 TFLOP/s of fp32 products, and 767 us, 336
//    TFLOP/s, in a replayed graph on the same inputs; three fp16 products at the measured matrix rate are 461 us.
//    One issuing thread for both products stood in its own way with heads of 64, whose products are short (a matrix
//    instruction takes about 45 cycles to issue): 124 us against 111.
//  Tiles that the parts cannot hold (NaN, infinities, magnitudes from 2^40 on; a key or value row whose largest element is
//  below 2^-14 of the tile's; nothing but values below 2^-40) are flagged by k_win_prep; a CTA that would read a flagged tile,
//  or has such a q, computes its rows with plain fp32 code that reads only what each row sees: a warp per row, one key after
//  another. Of the 16384 rows above, one such tile of one key-value head in the middle makes it 16 ms, the first tokens' tile of
//  one head 59 ms, of all four 197 ms.
// Every wait is bounded; a timeout records KX_STATUS_TIMEOUT in the status word and the CTA stops: its rows are left as they
// were, or, where a block is split, become NaN.
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
constexpr int WN_KEYS = 64;    // keys per tile
constexpr int WN_ROWS = 128;   // rows per CTA
constexpr int WN_GROUP = 128;  // threads of a softmax group
constexpr int WN_THREADS = 3 * WN_GROUP;
// registers per thread: launched with 168 (384 x 168 = 64,512); the two softmax groups take 232, the third warpgroup, of
// which two threads fetch and issue, keeps 40: 256 x 232 + 128 x 40 = 64,512
constexpr int WN_DMAX = 128;
constexpr float WN_HUGE = 1099511627776.0f;  // 2^40
// value tiles' scales go no lower, so that the factor of P.V (the scale, 2^-53 at least, times a tile's share) is a normal
// number for every share that can show next to others
constexpr int WN_LOW = -40;
// A row's output and sum are relative to a score that its largest may pass by this (in base 2) before they are scaled to
// it: fp32 has the room, and tiles that scale nothing save a pass over the output.
constexpr float WN_SLACK = 16.0f;
constexpr float WN_TINY = 9.094947e-13f;     // 2^-40
constexpr float WN_RANGE = 16384.0f;         // 2^14: the rows of a tile keep 2^-24 of their own largest value
// Scores (in base 2) from here on are rounded before the maximum is taken off, as the maximum is: the unrounded product
// less the rounded maximum is off by half a unit of the score, which for scores of 2^25 and more carries p out of fp16's
// range either way (NaN, or rows of zeros). Below, it is off by 2^-4 at most.
constexpr float WN_FAR = 1048576.0f;         // 2^20

struct WinArgs {
    const float *q, *k, *v;
    float* ctx;
    const int32_t *q_len, *k_len;
    uint8_t* ws;
    int* status;
    int ldq, ldk, ldv, ldc, B, Rq, S, H, Hkv, dk, dv, window, sinks;
    int G, chunks, per_chunk;  // query heads per key-value head, groups of them, heads per group (<= 128)
    int tiles;                 // of 64 keys in S
    int ka, vp;                // K planes of 64 x 64; value columns rounded up to 16
    int qt, qtiles;            // queries per block of rows, blocks per sample and group
    int splits;                // CTAs per block of rows, each with a part of its tiles
    size_t parts;              // where in the workspace their results are
    uint32_t block;            // bytes per tile of the workspace
    float scale2;
    bool vecq, veck, vecv;
};

// a tile's block: K high planes, K low planes, V^T high, V^T low; behind the last block one TileInfo per tile
struct alignas(16) TileInfo {
    float kscale, vscale;  // what products of its keys, its values are multiplied with
    int plain;             // it holds values that the parts cannot
    int pad;
};
__host__ __device__ inline uint32_t k_bytes(int ka) { return static_cast<uint32_t>(ka) * 2 * 8192; }
__host__ __device__ inline uint32_t v_bytes(int vp) { return static_cast<uint32_t>(vp) * 256; }

__device__ __forceinline__ TileInfo* infos(const WinArgs& A) {
    return reinterpret_cast<TileInfo*>(A.ws + static_cast<size_t>(A.B) * A.Hkv * A.tiles * A.block);
}

__device__ __forceinline__ bool sample_lens(const WinArgs& A, int b, int* q, int* k) {
    *q = A.q_len ? A.q_len[b] : A.Rq;
    *k = A.k_len ? A.k_len[b] : A.S;
    return *q >= 0 && *q <= A.Rq && *k >= 0 && *k <= A.S;
}

// the tiles that hold keys seen from a position in [p0, p1]: 0 .. na - 1 (first tokens), b0 .. end - 1
struct Tiles {
    int na, b0, end;
    __device__ __forceinline__ int count() const { return na + end - b0; }
    __device__ __forceinline__ int at(int i) const { return i < na ? i : b0 + i - na; }
};
// a block of WN_ROWS rows: queries i0 .. of a sample, the heads of a group
struct Block {
    int b, kvh, head0, heads, i0;
    __device__ __forceinline__ Block(const WinArgs& A, int index) {  // later queries see more keys: they come first
        const int per = A.B * A.Hkv * A.chunks, x = index % per, chunk = x % A.chunks, bh = x / A.chunks;
        b = bh / A.Hkv;
        kvh = bh - b * A.Hkv;
        head0 = kvh * A.G + chunk * A.per_chunk;
        heads = min(A.per_chunk, A.G - chunk * A.per_chunk);
        i0 = (A.qtiles - 1 - index / per) * A.qt;
    }
};
// A CTA's part of a split block: per row maximum and sum, then the rows' outputs, not divided yet; the first CTA's also
// says whether there is something to join.
constexpr int WN_MAX_PARTS = 224;
struct alignas(16) PartHead {
    int join, pad[3];
    float2 ml[WN_ROWS];
};
__host__ __device__ inline size_t part_bytes(int dv) { return sizeof(PartHead) + static_cast<size_t>(WN_ROWS) * ((dv + 3) / 4 * 4) * 4; }
__device__ __forceinline__ Tiles tiles_of(const WinArgs& A, int p0, int p1) {
    Tiles t{0, 0, 0};
    if (p1 < 0) return t;
    // max: the first of very many queries may lie 2^31 before the first key
    const int w0 = A.window > 0 ? max(0, max(p0, 0) - A.window + 1) : 0, s0 = min(A.sinks, w0);
    t.na = (s0 + WN_KEYS - 1) / WN_KEYS;
    t.b0 = max(t.na, w0 / WN_KEYS);
    t.end = p1 / WN_KEYS + 1;
    return t;
}

// x = (hi + lo), two fp16 each of a pair
__device__ __forceinline__ void parts2(float a, float b, uint32_t* hi, uint32_t* lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    const float2 rest = kx::fma2(f, make_float2(-1.0f, -1.0f), make_float2(a, b));
    const __half2 l = __floats2half2_rn(rest.x, rest.y);
    *hi = *reinterpret_cast<const uint32_t*>(&h);
    *lo = *reinterpret_cast<const uint32_t*>(&l);
}
// the power of two that brings `top` (the largest magnitude) into [2^13, 2^14), and its inverse
// (top < 2^40; what is below 2^lowest keeps its distance to that: scores of q or keys below 2^-100 are as good as zero, and
// value tiles below 2^WN_LOW go the plain way)
__device__ __forceinline__ float scale_up(float top, int lowest, float* down) {
    const int e = min(max(static_cast<int>(__float_as_uint(top) >> 23) - 127, lowest), 40);
    *down = __uint_as_float(static_cast<uint32_t>(127 - 13 + e) << 23);
    return __uint_as_float(static_cast<uint32_t>(127 + 13 - e) << 23);
}
// byte of 16-byte chunk c of row r in a 128-byte-swizzled plane
__device__ __forceinline__ uint32_t swz(int r, int c) { return static_cast<uint32_t>(r * 128 + ((c ^ (r & 7)) << 4)); }

__device__ __forceinline__ float4 load4(const float* p, int d, int n, bool vec) {  // elements d .. d + 3 of n, 0 behind them
    if (vec && d + 3 < n) return *reinterpret_cast<const float4*>(p + d);
    return make_float4(d < n ? p[d] : 0.f, d + 1 < n ? p[d + 1] : 0.f, d + 2 < n ? p[d + 2] : 0.f, d + 3 < n ? p[d + 3] : 0.f);
}
__device__ __forceinline__ float top4(float m, float4 x) {
    return fmaxf(m, fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))));
}
__device__ __forceinline__ bool held(float x) { return fabsf(x) < WN_HUGE; }  // false for NaN
__device__ __forceinline__ bool held4(float4 x) { return held(x.x) && held(x.y) && held(x.z) && held(x.w); }

// Bound: HBM and L2 writes, 4 bytes read and 4 written per element. A CTA per tile: both operands into shared memory,
// their largest magnitudes, then the parts in whole 128-byte rows of the swizzled planes.
__global__ void __launch_bounds__(256) k_win_prep(const __grid_constant__ WinArgs A) {
    extern __shared__ float rows[];  // K, then V: 64 rows of 129
    __shared__ float tops[2][8];
    constexpr int P = WN_DMAX + 1;
    float *ks = rows, *vs = rows + WN_KEYS * P;
    kx::griddep_wait();
    kx::griddep_launch_dependents();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int tile = blockIdx.x % A.tiles, bh = blockIdx.x / A.tiles, b = bh / A.Hkv, h = bh - b * A.Hkv;
    int ql, kl;
    if (!sample_lens(A, b, &ql, &kl)) return;
    const int j0 = tile * WN_KEYS, n = min(WN_KEYS, kl - j0);
    if (n <= 0 || ql == 0) return;
    {  // seen by no query
        const Tiles t = tiles_of(A, kl - ql, kl - 1);
        if (tile >= t.na && tile < t.b0) return;
    }
    bool good = true;
    float ktop = 0.0f, vtop = 0.0f, krow[WN_KEYS / 8], vrow[WN_KEYS / 8];
    const float* kr = A.k + (static_cast<long>(b) * A.S + j0) * A.ldk + h * A.dk;
    const float* vr = A.v + (static_cast<long>(b) * A.S + j0) * A.ldv + h * A.dv;
    // a warp per row, all of its rows asked for at once; rows behind the last key and rows that no query sees (behind the
    // first tokens, before the first query's window) are zero, so that they touch neither the scales nor the flag
    const int back = max(kl - ql, 0) - A.window;  // the last position before every window
    float4 kx4[WN_KEYS / 8], vx4[WN_KEYS / 8];
#pragma unroll
    for (int u = 0; u < WN_KEYS / 8; u++) {
        const int r = warp + 8 * u;
        kx4[u] = vx4[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < n && (A.window <= 0 || j0 + r > back || j0 + r < A.sinks)) {
            kx4[u] = load4(kr + static_cast<long>(r) * A.ldk, lane * 4, A.dk, A.veck);
            vx4[u] = load4(vr + static_cast<long>(r) * A.ldv, lane * 4, A.dv, A.vecv);
        }
    }
#pragma unroll
    for (int u = 0; u < WN_KEYS / 8; u++) {
        const int r = warp + 8 * u;
        const float4 x = kx4[u], y = vx4[u];
        good = good && held4(x) && held4(y);
        krow[u] = top4(0.0f, x);
        vrow[u] = top4(0.0f, y);
        float *kd = ks + r * P + lane * 4, *vd = vs + r * P + lane * 4;
        kd[0] = x.x, kd[1] = x.y, kd[2] = x.z, kd[3] = x.w;
        vd[0] = y.x, vd[1] = y.y, vd[2] = y.z, vd[3] = y.w;
    }
    // the rows' largest magnitudes, then the tile's
#pragma unroll
    for (int u = 0; u < WN_KEYS / 8; u++) {
#pragma unroll
        for (int d = 16; d; d >>= 1) {
            krow[u] = fmaxf(krow[u], __shfl_xor_sync(FULL, krow[u], d));
            vrow[u] = fmaxf(vrow[u], __shfl_xor_sync(FULL, vrow[u], d));
        }
        ktop = fmaxf(ktop, krow[u]);
        vtop = fmaxf(vtop, vrow[u]);
    }
    if (lane == 0) {
        tops[0][warp] = ktop;
        tops[1][warp] = vtop;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; w++) {
        ktop = fmaxf(ktop, tops[0][w]);
        vtop = fmaxf(vtop, tops[1][w]);
    }
    // a row far below the tile's largest would lose bits to its neighbour, which its query may not even see
#pragma unroll
    for (int u = 0; u < WN_KEYS / 8; u++)
        good = good && (krow[u] == 0.0f || krow[u] * WN_RANGE >= ktop) && (vrow[u] == 0.0f || vrow[u] * WN_RANGE >= vtop);
    good = good && (vtop == 0.0f || vtop >= WN_TINY);
    good = __syncthreads_and(good);
    float kdown, vdown;
    const float kup = scale_up(ktop, -100, &kdown), vup = scale_up(vtop, WN_LOW, &vdown);
    uint8_t* out = A.ws + static_cast<size_t>(blockIdx.x) * A.block;
    // K: chunk c of 8 head dims of key r; eight threads write a plane's row
    for (int x = tid; x < WN_KEYS * 8 * A.ka; x += 256) {
        const int c = x & 7, r = (x >> 3) & (WN_KEYS - 1), plane = x >> 9;
        const float* src = ks + r * P + plane * 64 + c * 8;
        uint4 hi, lo;
        uint32_t *hw = &hi.x, *lw = &lo.x;
#pragma unroll
        for (int e = 0; e < 4; e++) parts2(src[2 * e] * kup, src[2 * e + 1] * kup, hw + e, lw + e);
        *reinterpret_cast<uint4*>(out + plane * 8192 + swz(r, c)) = hi;
        *reinterpret_cast<uint4*>(out + (A.ka + plane) * 8192 + swz(r, c)) = lo;
    }
    // V transposed: chunk c of 8 keys of head dim d
    out += k_bytes(A.ka);
    for (int x = tid; x < A.vp * 8; x += 256) {
        const int c = x & 7, d = x >> 3;
        const float* src = vs + c * 8 * P + d;
        uint4 hi, lo;
        uint32_t *hw = &hi.x, *lw = &lo.x;
#pragma unroll
        for (int e = 0; e < 4; e++) parts2(src[2 * e * P] * vup, src[(2 * e + 1) * P] * vup, hw + e, lw + e);
        *reinterpret_cast<uint4*>(out + swz(d, c)) = hi;
        *reinterpret_cast<uint4*>(out + A.vp * 128 + swz(d, c)) = lo;
    }
    if (tid == 0) infos(A)[blockIdx.x] = TileInfo{kdown, vdown, !good, 0};
}
constexpr int WN_PREP_SMEM = 2 * WN_KEYS * (WN_DMAX + 1) * 4;

template <int D>
struct Win {
    static constexpr int KB = D / 64 * 2 * 8192, VB = D * 256;  // bytes of a K and a V tile, at most; three of each
    // K and V tiles 0 and 1, K tile 2, V tile 2: q's rows as they come lie from K tile 2 on
    static constexpr int V0 = 2 * KB, K2 = V0 + 2 * VB, V2 = K2 + KB, TOPS = V2 + VB, SMEM = TOPS + 2 * WN_ROWS * 4 + 1024;
    // tensor memory columns: q's high and low parts, NS tiles' S (P over it), P.V of either group. With a third S a group
    // that has stored P finds its next tile's S and may leave P.V to be added later; head dims above 64 leave no room
    // for it (with q's low parts in shared memory they would, but those products then take half as long again: 210 us
    // against 179 for 4096 rows). A third group for heads up to 64, with 152 registers per thread: 136 us against 108.
    static constexpr int NS = D > 64 ? 2 : 3;
    static constexpr bool AHEAD = NS == 3;
    static constexpr uint32_t TQH = 0, TQL = D / 2, TS = D, TO = 256, COLS = 512;
    static_assert(TS + NS * WN_KEYS <= TO && TO + 2 * D <= COLS, "tensor memory");
    static_assert(K2 + WN_ROWS * D * 4 <= TOPS, "q's rows fit");
    static_assert(TOPS >= WN_ROWS * (D + 2 + 4) * 4, "the groups' halves, maxima and sums fit in the tiles' place");
    __device__ __forceinline__ static int k_at(int s) { return s < 2 ? s * KB : K2; }
    __device__ __forceinline__ static int v_at(int s) { return s < 2 ? V0 + s * VB : V2; }
};

struct WinCtl {
    uint64_t kfull[3], kfree[3], vfull[3], vfree[3];  // tiles in shared memory
    uint64_t sfull[3], sfree[3];                      // S computed, P over it used
    uint64_t pready[2], ofull[2];                     // per group: P stored, P.V computed
    uint64_t drained[2];                              // after a timeout: an issuer's matrix instructions have ended
    uint32_t tmem;
    int abort, slow;
};

// The rows of a CTA in plain fp32, a warp per row: lanes over the head dims, one key after another. For inputs that the
// parts cannot hold; reads no key that the row does not see.
__device__ __noinline__ void plain_rows(const WinArgs& A, int b, int kvh, int head0, int heads, int i0, int rows, int off, int warp,
                                        int warps) {
    const int lane = threadIdx.x & 31;
    for (int r = warp; r < rows; r += warps) {
        const int i = i0 + r / heads, h = head0 + r % heads, p = off + i;
        const float* qr = A.q + (static_cast<long>(b) * A.Rq + i) * A.ldq + static_cast<long>(h) * A.dk;
        float q[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int x = 0; x < 4; x++) q[x] = lane + 32 * x < A.dk ? qr[lane + 32 * x] * A.scale2 : 0.0f;
        const int w0 = A.window > 0 ? max(0, p - A.window + 1) : 0, s0 = min(A.sinks, w0);
        // weights up to 2^off: below 1 / (p + 1), so that no sum of weighted values passes the largest value
        const float off = static_cast<float>(__clz(p + 1) - 32);
        for (int j = s0 > 0 ? 0 : w0; j <= p; j = j + 1 == s0 ? w0 : j + 1) {
            const float* kr = A.k + (static_cast<long>(b) * A.S + j) * A.ldk + kvh * A.dk;
            const float* vr = A.v + (static_cast<long>(b) * A.S + j) * A.ldv + kvh * A.dv;
            float s = 0.0f;
#pragma unroll
            for (int x = 0; x < 4; x++)
                if (lane + 32 * x < A.dk) s = fmaf(q[x], kr[lane + 32 * x], s);
#pragma unroll
            for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(FULL, s, d);
            // a NaN score stays: it makes the sum NaN
            const float mn = fmaxf(m, s), safe = mn == -INFINITY ? 0.0f : mn;
            const float back = m == mn ? 1.0f : kx::ex2_approx(m - safe), e = kx::ex2_approx((s - safe) + off);
            m = mn;
            l = l * back + e;
#pragma unroll
            for (int x = 0; x < 4; x++)
                if (lane + 32 * x < A.dv) o[x] = o[x] * back + e * vr[lane + 32 * x];
        }
        float* out = A.ctx + (static_cast<long>(b) * A.Rq + i) * A.ldc + static_cast<long>(h) * A.dv;
#pragma unroll
        for (int x = 0; x < 4; x++)
            if (lane + 32 * x < A.dv) out[lane + 32 * x] = l == 0.0f ? 0.0f : o[x] / l;
    }
}

// SPLIT: a block's tiles over A.splits CTAs
template <int D, bool SPLIT>
__global__ void __launch_bounds__(WN_THREADS, 1) k_win_main(const __grid_constant__ WinArgs A) {
    using W = Win<D>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ WinCtl ctl;
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int splits = SPLIT ? A.splits : 1;
    const int block = static_cast<int>(blockIdx.x) / splits, split = static_cast<int>(blockIdx.x) - block * splits;
    const Block at(A, block);
    const int b = at.b, kvh = at.kvh, head0 = at.head0, heads = at.heads, i0 = at.i0, bh = b * A.Hkv + kvh;

    if (tid == 0) {
        for (int s = 0; s < 3; s++) {
            kx::mbar_init(&ctl.kfull[s], 1);
            kx::mbar_init(&ctl.kfree[s], 1);
            kx::mbar_init(&ctl.sfull[s], 1);
            kx::mbar_init(&ctl.sfree[s], 1);
            kx::mbar_init(&ctl.vfull[s], 1);
            kx::mbar_init(&ctl.vfree[s], 1);
        }
        for (int g = 0; g < 2; g++) {
            kx::mbar_init(&ctl.pready[g], WN_GROUP);
            kx::mbar_init(&ctl.ofull[g], 1);
        }
        kx::mbar_init(&ctl.drained[0], 1);
        kx::mbar_init(&ctl.drained[1], 1);
        ctl.abort = 0;
        ctl.slow = 0;
        kx::fence_mbar_init();
    }
    if (warp == 8) {
        kx::tmem_alloc(&ctl.tmem, W::COLS);
        kx::tmem_relinquish();
    }
    kx::tc_fence_before();
    __syncthreads();
    kx::tc_fence_after();
    const uint32_t tmem = ctl.tmem;
    kx::griddep_wait();
    if (SPLIT) kx::griddep_launch_dependents();

    int ql, kl;
    const bool lens_ok = sample_lens(A, b, &ql, &kl);
    const int nq = lens_ok ? max(0, min(A.qt, ql - i0)) : 0, rows = nq * heads, off = kl - ql;
    if (!lens_ok) {  // NaN rows, reported
        if (tid == 0) kx::kv_report(A.status, KX_STATUS_BAD_REQUEST);
        const int nr = min(A.qt, A.Rq - i0);
        for (int y = tid; y < nr * heads * A.dv; y += WN_THREADS) {
            const int d = y % A.dv, r = y / A.dv;
            A.ctx[(static_cast<long>(b) * A.Rq + i0 + r / heads) * A.ldc + static_cast<long>(head0 + r % heads) * A.dv + d] = NAN;
        }
    }
    Tiles tl{0, 0, 0};
    if (nq > 0) tl = tiles_of(A, off + i0, off + i0 + nq - 1);
    const int all_tiles = tl.count(), t0 = static_cast<int>(static_cast<long>(all_tiles) * split / splits);
    const int n_tiles = static_cast<int>(static_cast<long>(all_tiles) * (split + 1) / splits) - t0;
    const int turn = tl.na - t0, before = t0, behind = tl.b0 - turn;  // this CTA's tile t: tl.at(t0 + t)
    const auto tile_at = [&](int t) { return t + (t < turn ? before : behind); };
    const auto part = [&] { return reinterpret_cast<PartHead*>(A.ws + A.parts + blockIdx.x * part_bytes(A.dv)); };
    const uint8_t* blocks = A.ws + static_cast<size_t>(bh) * A.tiles * A.block;
    const TileInfo* info = infos(A) + static_cast<size_t>(bh) * A.tiles;

    // K (warp 8) and V (warp 10) of tile t into their places
    const auto fetch_k = [&](int t) {
        const int s = t % 3;
        if (t >= 3 && !kx::mbar_wait(&ctl.kfree[s], (t / 3 - 1) & 1, &ctl.abort, A.status)) return false;
        kx::mbar_arrive_expect_tx(&ctl.kfull[s], k_bytes(A.ka));
        kx::bulk_load(smem + W::k_at(s), blocks + static_cast<size_t>(tile_at(t)) * A.block, k_bytes(A.ka), &ctl.kfull[s]);
        return true;
    };
    const auto fetch_v = [&](int t) {
        const int s = t % 3;
        if (t >= 3 && !kx::mbar_wait(&ctl.vfree[s], (t / 3 - 1) & 1, &ctl.abort, A.status)) return false;
        kx::mbar_arrive_expect_tx(&ctl.vfull[s], v_bytes(A.vp));
        kx::bulk_load(smem + W::v_at(s), blocks + static_cast<size_t>(tile_at(t)) * A.block + k_bytes(A.ka), v_bytes(A.vp), &ctl.vfull[s]);
        return true;
    };
    constexpr int EARLY = 2;  // tiles fetched while q is prepared (K's third place is lent to q until then)
    if (warp == 8 && lane == 0)
        for (int t = 0; t < min(n_tiles, EARLY); t++) fetch_k(t);
    if (warp == 10 && lane == 0)
        for (int t = 0; t < min(n_tiles, EARLY); t++) fetch_v(t);

    // q's parts: group g takes the head dims [g D / 2, (g + 1) D / 2) of row r
    const int grp = warp >> 2, r = tid & (WN_ROWS - 1);
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const int my_i = r / heads, my_p = r < rows ? off + i0 + my_i : -1;
    float cs = 0.0f;  // what a score's products are multiplied with, besides the tile's scale
    if (grp < 2 && nq > 0) {
        bool slow = false;
        // rows in order into shared memory, chunk y of row x at place y ^ (x & 7); from there every thread takes its half row
        float4* stage = reinterpret_cast<float4*>(smem + W::K2);
        float* tops = reinterpret_cast<float*>(smem + W::TOPS);
        constexpr int STEP = 2 * WN_GROUP / (D / 4);  // rows at a time
        const int y = tid % (D / 4), di = STEP / heads, dh = STEP - di * heads;
        int i = tid / (D / 4) / heads, h = tid / (D / 4) - i * heads;
#pragma unroll 4
        for (int x = tid / (D / 4); x < WN_ROWS; x += STEP) {
            const float* qr = A.q + (static_cast<long>(b) * A.Rq + i0 + i) * A.ldq + static_cast<long>(head0 + h) * A.dk;
            float4* to = stage + x * (D / 4) + (y ^ (x & 7));
            if (A.vecq) {
                const bool in = x < rows && y * 4 < A.dk;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                             ::"r"(kx::smem_u32(to)), "l"(in ? qr + y * 4 : A.q), "r"(in ? 16 : 0)
                             : "memory");
            } else {
                *to = x < rows ? load4(qr, y * 4, A.dk, false) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
            i += di, h += dh;
            if (h >= heads) h -= heads, i++;
        }
        for (int t = tid; t < all_tiles; t += 2 * WN_GROUP) slow = slow || __ldcg(&info[tl.at(t)].plain) != 0;
        asm volatile("cp.async.wait_all;" ::: "memory");
        kx::named_bar(1, 2 * WN_GROUP);
        float4 f[D / 8];
        float top = 0.0f;
#pragma unroll
        for (int y = 0; y < D / 8; y++) {
            f[y] = stage[r * (D / 4) + ((grp * (D / 8) + y) ^ (r & 7))];
            slow = slow || !held4(f[y]);
            top = top4(top, f[y]);
        }
        tops[grp * WN_ROWS + r] = top;
        if (slow) ctl.slow = 1;
        kx::named_bar(1, 2 * WN_GROUP);
        float down;
        float up = scale_up(fmaxf(tops[r], tops[WN_ROWS + r]), -100, &down);
        cs = down * fabsf(A.scale2);
        if (A.scale2 < 0.0f) up = -up;
#pragma unroll
        for (int y = 0; y < D / 8; y += 8) {
            uint32_t hi[16], lo[16];
#pragma unroll
            for (int z = 0; z < 8; z++) {
                parts2(f[y + z].x * up, f[y + z].y * up, hi + 2 * z, lo + 2 * z);
                parts2(f[y + z].z * up, f[y + z].w * up, hi + 2 * z + 1, lo + 2 * z + 1);
            }
            kx::tmem_st16(tmem + lanes + W::TQH + grp * (D / 4) + y * 2, hi);
            kx::tmem_st16(tmem + lanes + W::TQL + grp * (D / 4) + y * 2, lo);
        }
        kx::tmem_st_wait();
        kx::fence_proxy_async_smem();  // q's place is next written by bulk copies
    }
    kx::tc_fence_before();
    __syncthreads();
    kx::tc_fence_after();
    const bool slow = ctl.slow != 0;
    const int n = slow ? 0 : n_tiles;
    if (SPLIT && tid == 0 && split == 0) part()->join = !slow && all_tiles > 0;
    if (slow && grp < 2 && split == 0) plain_rows(A, b, kvh, head0, heads, i0, rows, off, warp, 8);

    if (grp == 2) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        if ((warp == 8 || warp == 10) && lane == 0) {  // fetch the tiles
            int sent = min(n_tiles, EARLY);
            bool good = true;
            for (; sent < n; sent++) {
                good = warp == 8 ? fetch_k(sent) : fetch_v(sent);
                if (!good) break;
            }
            // no copy may be under way when the CTA ends; where everything went well its last reader has seen to that
            if (slow || !good || ctl.abort) {
                const uint64_t t0 = kx::globaltimer();
                uint64_t* full = warp == 8 ? ctl.kfull : ctl.vfull;
                for (int t = max(0, sent - 3); t < sent; t++)
                    while (!kx::mbar_try_wait(&full[t % 3], (t / 3) & 1) && kx::globaltimer() - t0 < KX_WAIT_NS) __nanosleep(256);
            }
        } else if (warp == 9 || warp == 11) {  // issue the matrix instructions: a warp keeps together, one lane issues
            const uint32_t tm = __shfl_sync(FULL, tmem, 0), base = __shfl_sync(FULL, kx::smem_u32(smem), 0);
            const auto wait = [&](uint64_t* bar, int parity) {
                return __all_sync(FULL, kx::mbar_wait(bar, parity & 1, &ctl.abort, A.status)) != 0;
            };
            bool good = true;
            if (warp == 9) {  // S of tile t, in the place of tile t - NS once P there has been used
                const uint32_t id = kx::idesc_f16(WN_ROWS, WN_KEYS), lo = static_cast<uint32_t>(A.ka) * (8192 >> 4);
                const int ksteps = (A.dk + 15) / 16;
                for (int t = 0; t < n; t++) {
                    const int s = t % 3, z = t % W::NS;
                    good = wait(&ctl.kfull[s], t / 3) && (t < W::NS || wait(&ctl.sfree[z], t / W::NS - 1));
                    if (!good) break;
                    kx::tc_fence_after();
                    const uint32_t d = tm + W::TS + z * WN_KEYS;
                    const uint64_t kh = kx::desc_sw128_kmajor(base + W::k_at(s));
                    if (kx::elect_one()) {
#pragma unroll
                        for (int k = 0; k < D / 16; k++) {
                            if (k >= ksteps) break;
                            const uint64_t b = kh + (k >> 2) * (8192 >> 4) + (k & 3) * (32 >> 4);
                            kx::mma_f16_ts(d, tm + W::TQL + k * 8, b, id, k != 0);
                            kx::mma_f16_ts(d, tm + W::TQH + k * 8, b + lo, id, 1);
                            kx::mma_f16_ts(d, tm + W::TQH + k * 8, b, id, 1);
                        }
                        kx::mma_commit(&ctl.sfull[z]);
                        kx::mma_commit(&ctl.kfree[s]);
                    }
                    __syncwarp();
                }
            } else {  // P.V of tile t; P: high parts of 32 keys, their low parts, and again
                const uint32_t id = kx::idesc_f16(WN_ROWS, A.vp), lo = static_cast<uint32_t>(A.vp) * (128 >> 4);
                for (int t = 0; t < n; t++) {
                    const int g = t & 1, s = t % 3, z = t % W::NS;
                    good = wait(&ctl.vfull[s], t / 3) && wait(&ctl.pready[g], t / 2);
                    if (!good) break;
                    kx::tc_fence_after();
                    const uint32_t a = tm + W::TS + z * WN_KEYS, d = tm + W::TO + g * D;
                    const uint64_t vh = kx::desc_sw128_kmajor(base + W::v_at(s));
                    if (kx::elect_one()) {
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            const uint32_t ph = a + (k >> 1) * 32 + (k & 1) * 8;
                            const uint64_t b = vh + k * (32 >> 4);
                            kx::mma_f16_ts(d, ph + 16, b, id, k != 0);
                            kx::mma_f16_ts(d, ph, b + lo, id, 1);
                            kx::mma_f16_ts(d, ph, b, id, 1);
                        }
                        kx::mma_commit(&ctl.ofull[g]);
                        kx::mma_commit(&ctl.sfree[z]);
                        kx::mma_commit(&ctl.vfree[s]);
                    }
                    __syncwarp();
                }
            }
            if (!good) {
                // matrix instructions may still be running: give them time to finish (bounded) before the tensor memory and
                // the shared memory go away
                uint64_t* bar = &ctl.drained[warp == 11];
                if (kx::elect_one()) kx::mma_commit(bar);
                const uint64_t t0 = kx::globaltimer();
                while (!kx::mbar_try_wait(bar, 0) && kx::globaltimer() - t0 < KX_WAIT_NS) __nanosleep(256);
            }
        }
        __syncwarp();
    } else {  // softmax groups
        asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
        float2 o[D / 2];  // the row's output so far and its sum l, relative to a score of m
        float m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int y = 0; y < D / 2; y++) o[y] = make_float2(0.0f, 0.0f);
        const uint32_t om = tmem + lanes + W::TO + grp * D;
        const int p_first = off + i0, p_last = off + i0 + nq - 1;
        float2 scales = make_float2(1.0f, 1.0f);  // a tile's, fetched a tile ahead
        if (grp < n) scales = __ldcg(reinterpret_cast<const float2*>(info + tile_at(grp)));
        float gain = 0.0f, gain_next = 0.0f;  // what P.V is multiplied with: its tile's scale and share
        const auto join = [&](int t) {  // P.V of tile t joins the output
            if (!__all_sync(FULL, kx::mbar_wait(&ctl.ofull[grp], (t / 2) & 1, &ctl.abort, A.status))) return false;
            kx::tc_fence_after();
#pragma unroll
            for (int c = 0; c < D; c += 32) {
                if (c >= A.vp) continue;
                uint32_t d[32];
                kx::tmem_ld32(om + c, d);
                kx::tmem_ld32_wait(d);
#pragma unroll
                for (int y = 0; y < 32; y += 2)
                    o[(c + y) / 2] = kx::fma2(make_float2(__uint_as_float(d[y]), __uint_as_float(d[y + 1])), make_float2(gain, gain),
                                              o[(c + y) / 2]);
            }
            kx::tc_fence_before();
            return true;
        };
        for (int t = grp; grp < n; t += 2) {
            float alpha = 1.0f;
            bool moved = false;  // m grows: what there is of the output shrinks by alpha
            if (t < n) {  // P of tile t
                const uint32_t sm = tmem + lanes + W::TS + (t % W::NS) * WN_KEYS;
                const int j0 = tile_at(t) * WN_KEYS;
                const float f = fmaxf(cs * scales.x, 1.17549435e-38f);  // positive: -inf stays -inf
                const float vscale = scales.y;
                if (t + 2 < n) scales = __ldcg(reinterpret_cast<const float2*>(info + tile_at(t + 2)));
                if (!__all_sync(FULL, kx::mbar_wait(&ctl.sfull[t % W::NS], (t / W::NS) & 1, &ctl.abort, A.status))) break;
                kx::tc_fence_after();
                // some row does not see some key of the tile
                const bool masked = j0 + WN_KEYS - 1 > p_first || !(A.window <= 0 || j0 > p_last - A.window || j0 + WN_KEYS <= A.sinks);
                const int from = A.window > 0 ? my_p - A.window - j0 : -1, to = my_p - j0, first = A.sinks - j0;
                const auto load = [&](int c, uint32_t(&x)[32]) {  // products with the keys 32 c .. 32 c + 31
                    kx::tmem_ld32(sm + c * 32, x);
                    kx::tmem_ld32_wait(x);
                    if (masked) {
#pragma unroll
                        for (int y = 0; y < 32; y++)
                            if (c * 32 + y > to || (c * 32 + y <= from && c * 32 + y >= first)) x[y] = 0xFF800000u;
                    }
                };
                uint32_t s[2][32];  // the second time for D > 64, whose output leaves no registers to keep both
                float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    uint32_t(&x)[32] = s[D > 64 ? 0 : c];
                    load(c, x);
#pragma unroll
                    for (int y = 0; y < 32; y++) top[y & 3] = fmaxf(top[y & 3], __uint_as_float(x[y]));
                }
                const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
                const float peak = __fmul_rn(mx, f), safe = peak == -INFINITY ? 0.0f : peak;
                if (peak > m + WN_SLACK) {
                    moved = m != -INFINITY;
                    alpha = kx::ex2_approx(m - peak);
                    m = peak;
                }
                const float share = kx::ex2_approx(peak - (m == -INFINITY ? 0.0f : m));
                const bool far = __any_sync(FULL, fabsf(safe) >= WN_FAR);
                const float mul = far ? 1.0f : f, shift = far ? 13.0f : 13.0f - safe;
                if (far) {
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        uint32_t(&x)[32] = s[D > 64 ? 0 : c];
                        if (D > 64) load(c, x);
#pragma unroll
                        for (int y = 0; y < 32; y++) x[y] = __float_as_uint(__fadd_rn(__fmul_rn(__uint_as_float(x[y]), f), -safe));
                        if (D > 64) kx::tmem_st32(sm + c * 32, x);
                    }
                    if (D > 64) kx::tmem_st_wait();
                }
                float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    uint32_t(&x)[32] = s[D > 64 ? 0 : c];
                    if (D > 64) load(c, x);
                    uint32_t hi[16], lo[16];
#pragma unroll
                    for (int y = 0; y < 32; y += 2) {
                        float2 e = kx::fma2(make_float2(__uint_as_float(x[y]), __uint_as_float(x[y + 1])), make_float2(mul, mul),
                                            make_float2(shift, shift));
                        e.x = kx::ex2_approx(e.x);
                        e.y = kx::ex2_approx(e.y);
                        sum[y / 2 & 1] = kx::add2(sum[y / 2 & 1], e);
                        parts2(e.x, e.y, hi + y / 2, lo + y / 2);
                    }
                    kx::tmem_st16(sm + c * 32, hi);
                    kx::tmem_st16(sm + c * 32 + 16, lo);
                }
                l = l * alpha + share * ((sum[0].x + sum[0].y) + (sum[1].x + sum[1].y));
                gain_next = share * vscale;
            }
            if (W::AHEAD && t >= 2 && !join(t - 2)) break;
            if (t >= n) break;
            if (__any_sync(FULL, moved)) {
#pragma unroll
                for (int y = 0; y < D / 2; y++) o[y] = kx::mul2(o[y], make_float2(alpha, alpha));
            }
            gain = gain_next;
            kx::tmem_st_wait();
            kx::tc_fence_before();
            kx::mbar_arrive(&ctl.pready[grp]);
            if (!W::AHEAD && !join(t)) break;
        }
        // the groups' rows through shared memory (the tiles' place: every matrix instruction that read them is done once both
        // groups have seen their last P.V): each joins one half of the columns, then whole rows are written
        if (n > 0) {
            constexpr int P = D / 2 + 1;
            float* half = reinterpret_cast<float*>(smem);  // [group that joins it][row][column]
            float* ml = half + 2 * WN_ROWS * P;            // [group][row]: what it is relative to, and the sum
            kx::named_bar(3, 2 * WN_GROUP);
            float* mine = ml + (grp * WN_ROWS + r) * 2;
            mine[0] = m, mine[1] = l;
            float* send = half + ((grp ^ 1) * WN_ROWS + r) * P;
#pragma unroll
            for (int x = 0; x < D / 4; x++) {
                const float2 v = grp == 0 ? o[D / 4 + x] : o[x];
                send[2 * x] = v.x, send[2 * x + 1] = v.y;
            }
            kx::named_bar(3, 2 * WN_GROUP);
            {
                const float* his = ml + ((grp ^ 1) * WN_ROWS + r) * 2;
                const float mm = fmaxf(m, his[0]), safe = mm == -INFINITY ? 0.0f : mm;
                float f0 = kx::ex2_approx(m - safe), f1 = kx::ex2_approx(his[0] - safe);
                const float den = f0 * l + f1 * his[1];
                // after a timeout the part's rows are not written: a sum of NaN makes the joined rows NaN
                if (SPLIT && grp == 0) part()->ml[r] = ctl.abort ? make_float2(0.0f, NAN) : make_float2(mm, den);
                const float inv = SPLIT ? 1.0f : den == 0.0f ? 0.0f : 1.0f / den;
                f0 *= inv, f1 *= inv;
                float* z = half + (grp * WN_ROWS + r) * P;
#pragma unroll
                for (int x = 0; x < D / 4; x++) {
                    const float2 v = grp == 0 ? o[x] : o[D / 4 + x];
                    z[2 * x] = f0 * v.x + f1 * z[2 * x];
                    z[2 * x + 1] = f0 * v.y + f1 * z[2 * x + 1];
                }
            }
            kx::named_bar(3, 2 * WN_GROUP);
            const int di = 8 / heads, dh = 8 - di * heads;
            int i = warp / heads, h = warp - i * heads;
            for (int x = warp; x < rows && !ctl.abort; x += 8) {
                float* out = SPLIT ? reinterpret_cast<float*>(part() + 1) + x * ((A.dv + 3) / 4 * 4)
                                          : A.ctx + (static_cast<long>(b) * A.Rq + i0 + i) * A.ldc + static_cast<long>(head0 + h) * A.dv;
#pragma unroll
                for (int c = 0; c < D; c += 32)
                    if (c + lane < A.dv) out[c + lane] = half[(c < D / 2 ? 0 : WN_ROWS * P) + x * P + c % (D / 2) + lane];
                i += di, h += dh;
                if (h >= heads) h -= heads, i++;
            }
        } else if (SPLIT && !slow && all_tiles > 0) {  // a split block with fewer tiles than parts
            if (grp == 0) part()->ml[r] = make_float2(-INFINITY, 0.0f);
        } else if (!slow && split == 0 && grp == 0 && r < rows) {  // rows that see nothing
            float* out = A.ctx + (static_cast<long>(b) * A.Rq + i0 + my_i) * A.ldc + static_cast<long>(head0 + r % heads) * A.dv;
            for (int y = 0; y < A.dv; y++) out[y] = 0.0f;
        }
    }
    kx::tc_fence_before();
    __syncthreads();
    if (warp == 8) {
        kx::tc_fence_after();
        kx::tmem_dealloc(tmem, W::COLS);
    }
}

// A warp per row of a split block, four elements per lane, the block's parts in their order, eight at a time. Everything is
// asked for before anything is looked at: the launch is one round trip to L2 where the parts are at most eight.
__global__ void __launch_bounds__(256) k_win_join(const __grid_constant__ WinArgs A) {
    kx::griddep_wait();
    kx::griddep_launch_dependents();
    const int block = blockIdx.x / (WN_ROWS / 8), r = blockIdx.x % (WN_ROWS / 8) * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int pitch = (A.dv + 3) / 4 * 4;
    const size_t bytes = part_bytes(A.dv);
    const uint8_t* parts = A.ws + A.parts + static_cast<size_t>(block) * A.splits * bytes;
    const int wanted = __ldcg(&reinterpret_cast<const PartHead*>(parts)->join);
    const Block at(A, block);
    int ql, kl;
    const bool lens_ok = sample_lens(A, at.b, &ql, &kl);
    float m = -INFINITY, den = 0.0f;
    float4 num = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s0 = 0; s0 < A.splits; s0 += 8) {
        float2 ml[8];
        float4 v[8];
#pragma unroll
        for (int u = 0; u < 8; u++) {
            const PartHead* p = reinterpret_cast<const PartHead*>(parts + min(s0 + u, A.splits - 1) * bytes);
            ml[u] = s0 + u < A.splits ? __ldcg(&p->ml[r]) : make_float2(-INFINITY, 0.0f);
            v[u] = s0 + u < A.splits && lane * 4 < pitch
                       ? __ldcg(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p + 1) + r * pitch + lane * 4))
                       : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        float top = m;
#pragma unroll
        for (int u = 0; u < 8; u++) top = fmaxf(top, ml[u].x);
        const float safe = top == -INFINITY ? 0.0f : top, back = kx::ex2_approx(m - safe);
        m = top;
        den *= back;
        num.x *= back, num.y *= back, num.z *= back, num.w *= back;
#pragma unroll
        for (int u = 0; u < 8; u++) {
            if (ml[u].x == -INFINITY) continue;  // that part saw nothing of the row: its output may not be there
            const float f = kx::ex2_approx(ml[u].x - safe);
            den += f * ml[u].y;
            num.x += f * v[u].x, num.y += f * v[u].y, num.z += f * v[u].z, num.w += f * v[u].w;
        }
    }
    // nothing to join (then the parts hold nothing, and what came of them is dropped), or behind the last row
    if (!wanted || !lens_ok || r >= min(A.qt, ql - at.i0) * at.heads) return;
    const float inv = den == 0.0f ? 0.0f : 1.0f / den;
    const int i = r / at.heads, h = r - i * at.heads;
    float* out = A.ctx + (static_cast<long>(at.b) * A.Rq + at.i0 + i) * A.ldc + static_cast<long>(at.head0 + h) * A.dv;
    const float z[4] = {num.x * inv, num.y * inv, num.z * inv, num.w * inv};
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (lane * 4 + e < A.dv) out[lane * 4 + e] = z[e];
}

struct WinLayout {
    int tiles, ka, vp;
    uint32_t block;
    size_t parts, bytes;
};
bool layout_of(int B, int S, int Hkv, int dk, int dv, WinLayout* L) {
    if (B < 0 || S < 1 || Hkv < 1 || dk < 1 || dv < 1 || dk > WN_DMAX || dv > WN_DMAX || S > INT32_MAX - 256) return false;
    L->tiles = (S + WN_KEYS - 1) / WN_KEYS;
    L->ka = (dk + 63) / 64;
    L->vp = (dv + 15) / 16 * 16;
    L->block = k_bytes(L->ka) + v_bytes(L->vp);
    const double blocks = static_cast<double>(B) * Hkv * L->tiles;
    if (blocks > 2e9) return false;
    L->parts = (static_cast<size_t>(B) * Hkv * L->tiles * (L->block + sizeof(TileInfo)) + 127) / 128 * 128;
    L->bytes = L->parts + WN_MAX_PARTS * part_bytes(dv);
    return true;
}

// more dynamic shared memory than the default: asked for once per device
int allow_smem(const void* kernel, int bytes, unsigned long long* devs_set) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return -1;
    const unsigned long long bit = 1ull << (dev & 63);
    if (__atomic_load_n(devs_set, __ATOMIC_ACQUIRE) & bit) return 0;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return -1;
    __atomic_fetch_or(devs_set, bit, __ATOMIC_RELEASE);
    return 0;
}

int launch_prep(const WinArgs& A, unsigned grid, cudaStream_t st) {
    static unsigned long long devs_set = 0;
    if (allow_smem(reinterpret_cast<const void*>(k_win_prep), WN_PREP_SMEM, &devs_set) != 0) return -1;
    return kx::launch_pdl(k_win_prep, dim3(grid), dim3(256), WN_PREP_SMEM, st, A);
}

template <int D, bool SPLIT>
int launch_main(const WinArgs& A, unsigned grid, cudaStream_t st) {
    static unsigned long long devs_set = 0;
    if (allow_smem(reinterpret_cast<const void*>(k_win_main<D, SPLIT>), Win<D>::SMEM, &devs_set) != 0) return -1;
    return kx::launch_pdl(k_win_main<D, SPLIT>, dim3(grid), dim3(WN_THREADS), Win<D>::SMEM, st, A);
}

}  // namespace

extern "C" {

size_t kx_attention_window_ws(int B, int S, int Hkv, int dk, int dv) {
    WinLayout L;
    return layout_of(B, S, Hkv, dk, dv, &L) ? L.bytes : 0;
}

int kx_attention_window(const float* q, int ldq, const float* k, int ldk, const float* v, int ldv, float* ctx, int ldc, int B, int Rq,
                        int S, int H, int Hkv, int dk, int dv, const int32_t* q_len, const int32_t* k_len, int window, int sinks,
                        float scale, void* ws, size_t ws_bytes, int* status, void* stream) {
    WinLayout L;
    if (!layout_of(B, S, Hkv, dk, dv, &L) || Rq < 0 || H < 1 || H % Hkv || sinks < 0 || !std::isfinite(scale * 1.4426950408889634f)) return -1;
    if (B == 0 || Rq == 0) return 0;
    if (!q || !k || !v || !ctx || ldq < static_cast<long>(H) * dk || ldk < static_cast<long>(Hkv) * dk ||
        ldv < static_cast<long>(Hkv) * dv || ldc < static_cast<long>(H) * dv)
        return -1;
    if (!ws || (reinterpret_cast<uintptr_t>(ws) & 127) || ws_bytes < L.bytes) return -1;
    WinArgs A;
    A.q = q, A.k = k, A.v = v, A.ctx = ctx, A.q_len = q_len, A.k_len = k_len;
    A.ws = static_cast<uint8_t*>(ws);
    A.status = status;
    A.ldq = ldq, A.ldk = ldk, A.ldv = ldv, A.ldc = ldc, A.B = B, A.Rq = Rq, A.S = S, A.H = H, A.Hkv = Hkv, A.dk = dk, A.dv = dv;
    // every position is below S: a window of S sees all there is (and no sum with it passes 32 bits)
    A.window = window >= S ? 0 : window, A.sinks = std::min(sinks, S);
    A.G = H / Hkv;
    A.chunks = (A.G + WN_ROWS - 1) / WN_ROWS;
    A.per_chunk = (A.G + A.chunks - 1) / A.chunks;
    A.chunks = (A.G + A.per_chunk - 1) / A.per_chunk;
    A.tiles = L.tiles, A.ka = L.ka, A.vp = L.vp, A.block = L.block;
    A.qt = WN_ROWS / A.per_chunk;
    A.qtiles = (Rq - 1) / A.qt + 1;
    A.scale2 = (scale == 0.0f ? 1.0f / sqrtf(static_cast<float>(dk)) : scale) * 1.4426950408889634f;
    const auto vec = [](const float* p, int ld, int d) { return ((ld | d) & 3) == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
    A.vecq = vec(q, ldq, dk), A.veck = vec(k, ldk, dk), A.vecv = vec(v, ldv, dv);
    const double blocks = static_cast<double>(A.qtiles) * B * Hkv * A.chunks;
    if (blocks > 2e9) return -1;
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0)
        return -1;
    // Two CTAs and more per block of rows where SMs would be idle otherwise: its tiles in as many parts, joined by a third
    // launch, at least four tiles (8 us) to a CTA. (Two parts each for 102 blocks on 148 SMs took 73 us against 58.)
    const int grid = static_cast<int>(blocks);
    const long reach = A.window > 0 ? std::min(static_cast<long>(S), static_cast<long>(A.window) + A.qt + A.sinks + 2 * WN_KEYS) : S;
    A.splits = static_cast<int>(std::min(static_cast<long>(sms / grid), reach / (4 * WN_KEYS)));
    if (A.splits < 2 || static_cast<long>(A.splits) * grid > WN_MAX_PARTS) A.splits = 1;
    A.parts = L.parts;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (launch_prep(A, static_cast<unsigned>(B * Hkv * L.tiles), st) != 0) return -1;
    const bool small = dk <= 64 && dv <= 64;
    if (A.splits == 1) return small ? launch_main<64, false>(A, grid, st) : launch_main<128, false>(A, grid, st);
    if ((small ? launch_main<64, true>(A, grid * A.splits, st) : launch_main<128, true>(A, grid * A.splits, st)) != 0) return -1;
    return kx::launch_pdl(k_win_join, dim3(static_cast<unsigned>(grid) * (WN_ROWS / 8)), dim3(256), 0, st, A);
}

}  // extern "C"
