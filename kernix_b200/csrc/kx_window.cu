// KERNIX-B200 attention of prompts with a sliding window whose first tokens stay visible (kx_attention_window,
// include/kx_kernels.h), in fp32, on the 5th-generation tensor cores. Per query row at position t and head, over the keys
// j <= t with j > t - window or j < sinks:  ctx = sum_j p_j v_j / sum_j p_j,  p_j = exp(s_j - max s),  s_j = scale q.k_j.
//
// fp32 accuracy from fp16 products: an fp32 value, scaled by a power of two so that the largest of its row is in
// [2^13, 2^14), is the sum of two fp16 parts up to 2^-22 of itself (up to 2^-39 of the row's largest where that is more),
// and a.b = ah.bh + al.bh + ah.bl: three fp16 products where 3xTF32 (the same 11-bit parts, no scaling) would cost six
// fp16 products' time. The scales are per query row, per key, and per 64 keys and value column, so that every
// accumulator has one scale; they are undone in fp32 (key scales before the softmax, value scales when a tile's p.v is
// added to the output). p in [0, 1] becomes p 2^13.
//
//  k_win_prep: per (sample, key-value head, tile of 64 keys) the parts of K (key-major) and V (transposed) in the
//    128-byte-swizzled layout that the matrix instructions read, one contiguous block, so that the main kernel fetches a
//    tile by two bulk copies and every CTA that reads it is spared the conversion. Tiles that no query sees are skipped.
//  k_win_main: one CTA per (sample, key-value head, 128 rows); a row is one query of one of the G heads that share the
//    keys (128 / G queries), so that few queries still fill the tile and a window's edges are short. Roles: a warp that
//    fetches tiles (ring of stages), a thread that issues the matrix instructions, and two groups of 128 threads, each
//    with every second tile: thread = row, S out of tensor memory, maximum, exponentials, P's parts back into tensor
//    memory over S (the A operand of P.V), then the tile's P.V added to the row's output in registers. While one group
//    works on its tile, the tensor cores work on the other's. Each group keeps a softmax of its own (maximum, sum,
//    output); the two are joined at the end.
//    Sums: S and a tile's P.V are at most 24 accumulated steps in the tensor core, everything longer is fp32 adds.
//  Values that the parts cannot hold (NaN, infinities, magnitudes from 2^60 on) are flagged per tile by k_win_prep; a CTA
//  that would read a flagged tile, or has such a q, computes its rows with plain fp32 code that reads only what each
//  row sees.
// Every wait is bounded; a timeout records KX_STATUS_TIMEOUT in the status word and the CTA stops.
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
// registers per thread: launched with 168 (384 x 168 = 64,512); the two softmax groups take 216, the third warpgroup, of
// which two threads fetch and issue, keeps 40: 256 x 216 + 128 x 40 = 60,416
constexpr int WN_DMAX = 128;
constexpr float WN_HUGE = 1152921504606846976.0f;  // 2^60

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
    int qt, qtiles;            // queries per CTA, CTAs per sample and group
    uint32_t block;            // bytes per tile of the workspace
    float scale2;
    bool vecq, veck, vecv, vecc;
};

// a tile's block: K high planes, K low planes, V^T high, V^T low, 64 key scales, vp value scales; the flags lie behind the
// last block
__host__ __device__ inline uint32_t k_bytes(int ka) { return static_cast<uint32_t>(ka) * 2 * 8192; }
__host__ __device__ inline uint32_t v_bytes(int vp) { return static_cast<uint32_t>(vp) * 256; }

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
__device__ __forceinline__ Tiles tiles_of(const WinArgs& A, int p0, int p1) {
    Tiles t{0, 0, 0};
    if (p1 < 0) return t;
    const int w0 = A.window > 0 ? max(0, p0 - A.window + 1) : 0, s0 = min(A.sinks, w0);
    t.na = (s0 + WN_KEYS - 1) / WN_KEYS;
    t.b0 = max(t.na, w0 / WN_KEYS);
    t.end = p1 / WN_KEYS + 1;
    return t;
}

// x = (hi + lo), two fp16 each of a pair
__device__ __forceinline__ void parts2(float a, float b, uint32_t* hi, uint32_t* lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
    *hi = *reinterpret_cast<const uint32_t*>(&h);
    *lo = *reinterpret_cast<const uint32_t*>(&l);
}
// the power of two that brings `top` (the largest magnitude) into [2^13, 2^14), and its inverse
__device__ __forceinline__ float scale_up(float top, float* down) {
    const int e = min(max(static_cast<int>(__float_as_uint(top) >> 23) - 127, -100), 126);
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

// Bound: HBM (and L2's write rate): 8 bytes read and 8 written per element pair of K and V.
__global__ void __launch_bounds__(256) k_win_prep(const __grid_constant__ WinArgs A) {
    __shared__ float vs[WN_KEYS][WN_DMAX + 1];
    __shared__ float part[8][WN_DMAX];
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
    uint8_t* out = A.ws + static_cast<size_t>(blockIdx.x) * A.block;
    float* kscale = reinterpret_cast<float*>(out + k_bytes(A.ka) + v_bytes(A.vp));
    float* vscale = kscale + WN_KEYS;
    bool good = true;
    // V into shared memory, and the columns' largest magnitudes
    for (int r = warp; r < WN_KEYS; r += 8) {
        const float* src = A.v + (static_cast<long>(b) * A.S + j0 + r) * A.ldv + h * A.dv;
        const float4 x = r < n ? load4(src, lane * 4, A.dv, A.vecv) : make_float4(0.f, 0.f, 0.f, 0.f);
        good = good && held4(x);
        vs[r][lane * 4] = x.x, vs[r][lane * 4 + 1] = x.y, vs[r][lane * 4 + 2] = x.z, vs[r][lane * 4 + 3] = x.w;
    }
    // K: a warp per row
    for (int r = warp; r < WN_KEYS; r += 8) {
        const float* src = A.k + (static_cast<long>(b) * A.S + j0 + r) * A.ldk + h * A.dk;
        const float4 x = r < n ? load4(src, lane * 4, A.dk, A.veck) : make_float4(0.f, 0.f, 0.f, 0.f);
        good = good && held4(x);
        float top = top4(0.0f, x);
#pragma unroll
        for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(FULL, top, d));
        float down;
        const float up = scale_up(top, &down);
        if (lane == 0) kscale[r] = down;
        uint2 hi, lo;
        parts2(x.x * up, x.y * up, &hi.x, &lo.x);
        parts2(x.z * up, x.w * up, &hi.y, &lo.y);
        const int plane = lane >> 4;  // 16 lanes x 4 elements = a plane's 64
        if (plane < A.ka) {
            uint8_t* to = out + plane * 8192 + swz(r, (lane & 15) >> 1) + (lane & 1) * 8;
            *reinterpret_cast<uint2*>(to) = hi;
            *reinterpret_cast<uint2*>(to + A.ka * 8192) = lo;
        }
    }
    good = __syncthreads_and(good);
    {  // column maxima: warp w over the keys 8 w .., then all
        for (int d = lane; d < A.vp; d += 32) {
            float top = 0.0f;
#pragma unroll
            for (int r = 0; r < 8; r++) top = fmaxf(top, fabsf(vs[warp * 8 + r][d]));
            part[warp][d] = top;
        }
        __syncthreads();
        for (int d = tid; d < A.vp; d += 256) {
            float top = 0.0f;
#pragma unroll
            for (int w = 0; w < 8; w++) top = fmaxf(top, part[w][d]);
            float down;
            part[0][d] = scale_up(top, &down);
            vscale[d] = down;
        }
        __syncthreads();
    }
    // V transposed: row d, 8 keys per 16-byte chunk
    uint8_t* vout = out + k_bytes(A.ka);
    for (int x = tid; x < A.vp * 8; x += 256) {
        const int d = x % A.vp, c = x / A.vp;
        const float up = part[0][d];
        uint4 hi, lo;
        uint32_t *hw = &hi.x, *lw = &lo.x;
#pragma unroll
        for (int e = 0; e < 4; e++) parts2(vs[c * 8 + 2 * e][d] * up, vs[c * 8 + 2 * e + 1][d] * up, hw + e, lw + e);
        *reinterpret_cast<uint4*>(vout + swz(d, c)) = hi;
        *reinterpret_cast<uint4*>(vout + A.vp * 128 + swz(d, c)) = lo;
    }
    if (tid == 0) reinterpret_cast<int*>(A.ws + static_cast<size_t>(A.B) * A.Hkv * A.tiles * A.block)[blockIdx.x] = !good;
}

template <int D>
struct Win {
    static constexpr int STAGES = 3;
    static constexpr int KB = D / 64 * 2 * 8192, VB = D * 256;  // bytes of a K and a V tile, at most
    static constexpr int SMEM = STAGES * (KB + VB) + 1024;
    // tensor memory columns: q's parts, then per group S (P over it) and P.V
    static constexpr uint32_t QH = 0, QL = D / 2, GRP = D, GRP_SIZE = WN_KEYS + D, COLS = 512;
    static_assert(GRP + 2 * GRP_SIZE <= COLS, "tensor memory");
    static_assert(STAGES * (KB + VB) >= WN_ROWS * (D + 1) * 4, "the second group's output fits in the stages");
};

struct WinCtl {
    uint64_t kfull[3], kfree[3], vfull[3], vfree[3];  // tiles in shared memory
    uint64_t sfull[2], pready[2], ofull[2];           // per group: S computed, P stored, P.V computed
    uint64_t drained;                                 // after a timeout: every matrix instruction has ended
    uint32_t tmem;
    int abort, slow;
    float qtop[2][WN_ROWS];
    alignas(16) float scales[2][2][WN_KEYS + WN_DMAX];  // per group, every other tile of it
    float ml[WN_ROWS][2];
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
            const float back = m == mn ? 1.0f : kx::ex2_approx(m - safe), e = kx::ex2_approx(s - safe);
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

template <int D>
__global__ void __launch_bounds__(WN_THREADS, 1) k_win_main(const __grid_constant__ WinArgs A) {
    using W = Win<D>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ WinCtl ctl;
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // later queries see more keys: their CTAs first
    const int per = A.B * A.Hkv * A.chunks;
    const int qi = A.qtiles - 1 - static_cast<int>(blockIdx.x) / per, x = static_cast<int>(blockIdx.x) % per;
    const int chunk = x % A.chunks, bh = x / A.chunks, b = bh / A.Hkv, kvh = bh - b * A.Hkv;
    const int head0 = kvh * A.G + chunk * A.per_chunk, heads = min(A.per_chunk, A.G - chunk * A.per_chunk);

    if (tid == 0) {
        for (int s = 0; s < W::STAGES; s++) {
            kx::mbar_init(&ctl.kfull[s], 1);
            kx::mbar_init(&ctl.kfree[s], 1);
            kx::mbar_init(&ctl.vfull[s], 1);
            kx::mbar_init(&ctl.vfree[s], 1);
        }
        for (int g = 0; g < 2; g++) {
            kx::mbar_init(&ctl.sfull[g], 1);
            kx::mbar_init(&ctl.pready[g], WN_GROUP);
            kx::mbar_init(&ctl.ofull[g], 1);
        }
        kx::mbar_init(&ctl.drained, 1);
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

    int ql, kl;
    const bool lens_ok = sample_lens(A, b, &ql, &kl);
    const int i0 = qi * A.qt, nq = lens_ok ? max(0, min(A.qt, ql - i0)) : 0, rows = nq * heads, off = kl - ql;
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
    const int n_tiles = tl.count();
    const uint8_t* blocks = A.ws + static_cast<size_t>(bh) * A.tiles * A.block;
    const int* flags = reinterpret_cast<const int*>(A.ws + static_cast<size_t>(A.B) * A.Hkv * A.tiles * A.block) + bh * A.tiles;

    // q's parts into tensor memory: group g takes the head dims [g D / 2, (g + 1) D / 2) of row r
    const int grp = warp >> 2, r = tid & (WN_ROWS - 1);
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const int my_i = r / heads, my_p = r < rows ? off + i0 + my_i : -1;
    float cs = 0.0f;  // what a score's products are multiplied with, besides the key's scale
    if (grp < 2 && nq > 0) {
        bool slow = false;
        for (int t = tid; t < n_tiles; t += 2 * WN_GROUP) slow = slow || __ldcg(flags + tl.at(t)) != 0;
        float4 f[D / 8];
        float top = 0.0f;
        const float* qr = A.q + (static_cast<long>(b) * A.Rq + i0 + my_i) * A.ldq + static_cast<long>(head0 + r % heads) * A.dk;
#pragma unroll
        for (int y = 0; y < D / 8; y++) {
            f[y] = r < rows ? load4(qr, grp * (D / 2) + y * 4, A.dk, A.vecq) : make_float4(0.f, 0.f, 0.f, 0.f);
            slow = slow || !held4(f[y]);
            top = top4(top, f[y]);
        }
        ctl.qtop[grp][r] = top;
        if (slow) ctl.slow = 1;
        kx::named_bar(1, 2 * WN_GROUP);
        float down;
        float up = scale_up(fmaxf(ctl.qtop[0][r], ctl.qtop[1][r]), &down);
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
            kx::tmem_st16(tmem + lanes + W::QH + grp * (D / 4) + y * 2, hi);
            kx::tmem_st16(tmem + lanes + W::QL + grp * (D / 4) + y * 2, lo);
        }
        kx::tmem_st_wait();
    }
    kx::tc_fence_before();
    __syncthreads();
    kx::tc_fence_after();
    const bool slow = ctl.slow != 0;
    const int n = slow ? 0 : n_tiles;
    if (slow && grp < 2) plain_rows(A, b, kvh, head0, heads, i0, rows, off, warp, 8);

    if (grp == 2) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        if (warp == 8 && lane == 0) {  // fetches the tiles
            bool ok = true;
            int sent = 0;
            for (int t = 0; t < n && ok; t++, sent++) {
                const int s = t % W::STAGES;
                const uint8_t* src = blocks + static_cast<size_t>(tl.at(t)) * A.block;
                uint8_t* dst = smem + s * (W::KB + W::VB);
                if (t >= W::STAGES) ok = kx::mbar_wait(&ctl.kfree[s], (t / W::STAGES - 1) & 1, &ctl.abort, A.status);
                if (!ok) break;
                kx::mbar_arrive_expect_tx(&ctl.kfull[s], k_bytes(A.ka));
                kx::bulk_load(dst, src, k_bytes(A.ka), &ctl.kfull[s]);
                if (t >= W::STAGES) ok = kx::mbar_wait(&ctl.vfree[s], (t / W::STAGES - 1) & 1, &ctl.abort, A.status);
                if (!ok) {  // this tile's K only
                    const uint64_t t0 = kx::globaltimer();
                    while (!kx::mbar_try_wait(&ctl.kfull[s], (t / W::STAGES) & 1) && kx::globaltimer() - t0 < KX_WAIT_NS) __nanosleep(256);
                    break;
                }
                kx::mbar_arrive_expect_tx(&ctl.vfull[s], v_bytes(A.vp));
                kx::bulk_load(dst + W::KB, src + k_bytes(A.ka), v_bytes(A.vp), &ctl.vfull[s]);
            }
            // no copy may still be under way when the CTA ends: the last ones issued complete every earlier one's phase too
            if (!ok || ctl.abort) {
                for (int t = max(0, sent - W::STAGES); t < sent; t++) {
                    const int s = t % W::STAGES;
                    const uint64_t t0 = kx::globaltimer();
                    while (!(kx::mbar_try_wait(&ctl.kfull[s], (t / W::STAGES) & 1) && kx::mbar_try_wait(&ctl.vfull[s], (t / W::STAGES) & 1)) &&
                           kx::globaltimer() - t0 < KX_WAIT_NS)
                        __nanosleep(256);
                }
            }
        } else if (warp == 9 && lane == 0) {  // issues the matrix instructions
            const uint32_t base = kx::smem_u32(smem);
            const uint32_t id_s = kx::idesc_f16(WN_ROWS, WN_KEYS), id_o = kx::idesc_f16(WN_ROWS, A.vp);
            const int ksteps = (A.dk + 15) / 16;
            bool ok = true;
            for (int t = 0; t <= n && ok; t++) {
                if (t < n) {  // S of tile t
                    const int g = t & 1, s = t % W::STAGES;
                    ok = kx::mbar_wait(&ctl.kfull[s], (t / W::STAGES) & 1, &ctl.abort, A.status);
                    // P of the group's tile before, which lies over S, has been used
                    if (ok && t >= 2) ok = kx::mbar_wait(&ctl.ofull[g], ((t - 2) / 2) & 1, &ctl.abort, A.status);
                    if (!ok) break;
                    kx::tc_fence_after();
                    const uint32_t d = tmem + W::GRP + g * W::GRP_SIZE, kh = base + s * (W::KB + W::VB), kl_ = kh + A.ka * 8192;
                    for (int k = 0; k < ksteps; k++) {
                        const uint32_t o = (k >> 2) * 8192 + (k & 3) * 32;
                        kx::mma_f16_ts(d, tmem + W::QL + k * 8, kx::desc_sw128_kmajor(kh + o), id_s, k != 0);
                        kx::mma_f16_ts(d, tmem + W::QH + k * 8, kx::desc_sw128_kmajor(kl_ + o), id_s, 1);
                        kx::mma_f16_ts(d, tmem + W::QH + k * 8, kx::desc_sw128_kmajor(kh + o), id_s, 1);
                    }
                    kx::mma_commit(&ctl.sfull[g]);
                    kx::mma_commit(&ctl.kfree[s]);
                }
                if (t >= 1) {  // P.V of tile t - 1; P: high parts of 32 keys, their low parts, and again
                    const int u = t - 1, g = u & 1, s = u % W::STAGES;
                    ok = kx::mbar_wait(&ctl.pready[g], (u / 2) & 1, &ctl.abort, A.status) &&
                         kx::mbar_wait(&ctl.vfull[s], (u / W::STAGES) & 1, &ctl.abort, A.status);
                    if (!ok) break;
                    kx::tc_fence_after();
                    const uint32_t p = tmem + W::GRP + g * W::GRP_SIZE, d = p + WN_KEYS;
                    const uint32_t vh = base + s * (W::KB + W::VB) + W::KB, vl = vh + A.vp * 128;
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const uint32_t ph = p + (k >> 1) * 32 + (k & 1) * 8, pl = ph + 16;
                        kx::mma_f16_ts(d, pl, kx::desc_sw128_kmajor(vh + k * 32), id_o, k != 0);
                        kx::mma_f16_ts(d, ph, kx::desc_sw128_kmajor(vl + k * 32), id_o, 1);
                        kx::mma_f16_ts(d, ph, kx::desc_sw128_kmajor(vh + k * 32), id_o, 1);
                    }
                    kx::mma_commit(&ctl.ofull[g]);
                    kx::mma_commit(&ctl.vfree[s]);
                }
            }
            if (!ok) {
                // matrix instructions may still be running: give them time to finish (bounded) before the tensor memory and
                // the shared memory go away
                kx::mma_commit(&ctl.drained);
                const uint64_t t0 = kx::globaltimer();
                while (!kx::mbar_try_wait(&ctl.drained, 0) && kx::globaltimer() - t0 < KX_WAIT_NS) __nanosleep(256);
            }
        }
        __syncwarp();
    } else {  // softmax groups
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        float o[D], m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int y = 0; y < D; y++) o[y] = 0.0f;
        const uint32_t sm = tmem + lanes + W::GRP + grp * W::GRP_SIZE;
        const int gt = tid & (WN_GROUP - 1), p_first = off + i0, p_last = off + i0 + nq - 1;
        float ks_next = 0.0f, vs_next = 0.0f;
        const auto fetch = [&](int t) {
            if (t >= n) return;
            const float* sc = reinterpret_cast<const float*>(blocks + static_cast<size_t>(tl.at(t)) * A.block + k_bytes(A.ka) + v_bytes(A.vp));
            if (gt < WN_KEYS) ks_next = __ldcg(sc + gt);
            if (gt < A.vp) vs_next = __ldcg(sc + WN_KEYS + gt);
        };
        bool ok = true;  // after a timeout the group still meets at its barriers
        fetch(grp);
        for (int t = grp; t < n; t += 2) {
            const int ph = (t / 2) & 1, j0 = tl.at(t) * WN_KEYS;
            float* scales = ctl.scales[grp][ph];
            if (gt < WN_KEYS) scales[gt] = ks_next;
            scales[WN_KEYS + gt] = vs_next;
            fetch(t + 2);
            kx::named_bar(1 + grp, WN_GROUP);
            ok = ok && __all_sync(FULL, kx::mbar_wait(&ctl.sfull[grp], ph, &ctl.abort, A.status));
            if (!ok) continue;
            kx::tc_fence_after();
            // every row sees every key of the tile
            const bool whole = j0 + WN_KEYS - 1 <= p_first &&
                               (A.window <= 0 || j0 > p_last - A.window || j0 + WN_KEYS <= A.sinks);
            const auto sees = [&](int j) { return j <= my_p && (A.window <= 0 || j > my_p - A.window || j < A.sinks); };
            float mx = -INFINITY;
#pragma unroll
            for (int c = 0; c < 2; c++) {
                uint32_t s[32];
                kx::tmem_ld32(sm + c * 32, s);
                kx::tmem_ld32_wait(s);
#pragma unroll
                for (int y = 0; y < 32; y += 4) {
                    const float4 ks = *reinterpret_cast<const float4*>(scales + c * 32 + y);
                    const float k4[4] = {ks.x, ks.y, ks.z, ks.w};
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float v = __uint_as_float(s[y + e]) * k4[e];
                        if (whole || sees(j0 + c * 32 + y + e)) mx = fmaxf(mx, v);
                    }
                }
            }
            const float mn = mx == -INFINITY ? m : fmaxf(m, mx * cs), safe = mn == -INFINITY ? 0.0f : mn, shift = 13.0f - safe;
            const float alpha = kx::ex2_approx(m - safe);
            m = mn;
            float sum = 0.0f;
#pragma unroll
            for (int c = 0; c < 2; c++) {
                uint32_t s[32], hi[16], lo[16];
                kx::tmem_ld32(sm + c * 32, s);
                kx::tmem_ld32_wait(s);
#pragma unroll
                for (int y = 0; y < 32; y += 4) {
                    const float4 ks = *reinterpret_cast<const float4*>(scales + c * 32 + y);
                    const float k4[4] = {ks.x, ks.y, ks.z, ks.w};
                    float p[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        p[e] = kx::ex2_approx(fmaf(__uint_as_float(s[y + e]) * k4[e], cs, shift));
                        if (!whole && !sees(j0 + c * 32 + y + e)) p[e] = 0.0f;
                        sum += p[e];
                    }
                    parts2(p[0], p[1], hi + y / 2, lo + y / 2);
                    parts2(p[2], p[3], hi + y / 2 + 1, lo + y / 2 + 1);
                }
                kx::tmem_st16(sm + c * 32, hi);
                kx::tmem_st16(sm + c * 32 + 16, lo);
            }
            l = l * alpha + sum;
            kx::tmem_st_wait();
            kx::tc_fence_before();
            kx::mbar_arrive(&ctl.pready[grp]);
            ok = __all_sync(FULL, kx::mbar_wait(&ctl.ofull[grp], ph, &ctl.abort, A.status));
            if (!ok) continue;
            kx::tc_fence_after();
#pragma unroll
            for (int c = 0; c < D; c += 32) {
                if (c >= A.vp) continue;
                uint32_t s[32];
                kx::tmem_ld32(sm + WN_KEYS + c, s);
                kx::tmem_ld32_wait(s);
#pragma unroll
                for (int y = 0; y < 32; y += 4) {
                    const float4 vsc = *reinterpret_cast<const float4*>(scales + WN_KEYS + c + y);
                    o[c + y] = fmaf(__uint_as_float(s[y]), vsc.x, o[c + y] * alpha);
                    o[c + y + 1] = fmaf(__uint_as_float(s[y + 1]), vsc.y, o[c + y + 1] * alpha);
                    o[c + y + 2] = fmaf(__uint_as_float(s[y + 2]), vsc.z, o[c + y + 2] * alpha);
                    o[c + y + 3] = fmaf(__uint_as_float(s[y + 3]), vsc.w, o[c + y + 3] * alpha);
                }
            }
            kx::tc_fence_before();
        }
        // the second group's rows through shared memory (the stages: every matrix instruction that read them is done once
        // both groups have seen their last P.V), then the first group writes
        if (n > 0) {
            float* other = reinterpret_cast<float*>(smem);
            kx::named_bar(3, 2 * WN_GROUP);
            if (grp == 1) {
                ctl.ml[r][0] = m;
                ctl.ml[r][1] = l;
#pragma unroll
                for (int y = 0; y < D; y++) other[r * (D + 1) + y] = o[y];
            }
            kx::named_bar(3, 2 * WN_GROUP);
            if (grp == 0 && r < rows && !ctl.abort) {
                const float m1 = ctl.ml[r][0], mm = fmaxf(m, m1), safe = mm == -INFINITY ? 0.0f : mm;
                const float f0 = kx::ex2_approx(m - safe), f1 = kx::ex2_approx(m1 - safe);
                const float den = f0 * l + f1 * ctl.ml[r][1], inv = den == 0.0f ? 0.0f : 1.0f / den;
                float* out = A.ctx + (static_cast<long>(b) * A.Rq + i0 + my_i) * A.ldc + static_cast<long>(head0 + r % heads) * A.dv;
#pragma unroll
                for (int y = 0; y < D; y += 4) {
                    float z[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) z[e] = (f0 * o[y + e] + f1 * other[r * (D + 1) + y + e]) * inv;
                    if (A.vecc && y + 3 < A.dv) {
                        *reinterpret_cast<float4*>(out + y) = make_float4(z[0], z[1], z[2], z[3]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (y + e < A.dv) out[y + e] = z[e];
                    }
                }
            }
        } else if (!slow && grp == 0 && r < rows) {  // rows that see nothing
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

struct WinLayout {
    int tiles, ka, vp;
    uint32_t block;
    size_t bytes;
};
bool layout_of(int B, int S, int Hkv, int dk, int dv, WinLayout* L) {
    if (B < 0 || S < 1 || Hkv < 1 || dk < 1 || dv < 1 || dk > WN_DMAX || dv > WN_DMAX || S > INT32_MAX - 256) return false;
    L->tiles = (S + WN_KEYS - 1) / WN_KEYS;
    L->ka = (dk + 63) / 64;
    L->vp = (dv + 15) / 16 * 16;
    L->block = (k_bytes(L->ka) + v_bytes(L->vp) + static_cast<uint32_t>(WN_KEYS + L->vp) * 4 + 127) / 128 * 128;
    const double blocks = static_cast<double>(B) * Hkv * L->tiles;
    if (blocks > 2e9) return false;
    L->bytes = static_cast<size_t>(B) * Hkv * L->tiles * (L->block + 4) + 16;
    return true;
}

template <int D>
int launch_main(const WinArgs& A, unsigned grid, cudaStream_t st) {
    static unsigned long long devs_set = 0;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return -1;
    const unsigned long long bit = 1ull << (dev & 63);
    if (!(__atomic_load_n(&devs_set, __ATOMIC_ACQUIRE) & bit)) {
        if (cudaFuncSetAttribute(k_win_main<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Win<D>::SMEM) != cudaSuccess) return -1;
        __atomic_fetch_or(&devs_set, bit, __ATOMIC_RELEASE);
    }
    return kx::launch_pdl(k_win_main<D>, dim3(grid), dim3(WN_THREADS), Win<D>::SMEM, st, A);
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
    if (!layout_of(B, S, Hkv, dk, dv, &L) || Rq < 0 || H < 1 || H % Hkv || sinks < 0 || !std::isfinite(scale)) return -1;
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
    A.window = window, A.sinks = sinks;
    A.G = H / Hkv;
    A.chunks = (A.G + WN_ROWS - 1) / WN_ROWS;
    A.per_chunk = (A.G + A.chunks - 1) / A.chunks;
    A.chunks = (A.G + A.per_chunk - 1) / A.per_chunk;
    A.tiles = L.tiles, A.ka = L.ka, A.vp = L.vp, A.block = L.block;
    A.qt = WN_ROWS / A.per_chunk;
    A.qtiles = (Rq + A.qt - 1) / A.qt;
    A.scale2 = (scale == 0.0f ? 1.0f / sqrtf(static_cast<float>(dk)) : scale) * 1.4426950408889634f;
    const auto vec = [](const float* p, int ld, int d) { return ((ld | d) & 3) == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
    A.vecq = vec(q, ldq, dk), A.veck = vec(k, ldk, dk), A.vecv = vec(v, ldv, dv), A.vecc = vec(ctx, ldc, dv);
    const double grid = static_cast<double>(A.qtiles) * B * Hkv * A.chunks;
    if (grid > 2e9) return -1;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (kx::launch_pdl(k_win_prep, dim3(static_cast<unsigned>(B * Hkv * L.tiles)), dim3(256), 0, st, A) != 0) return -1;
    return dk <= 64 && dv <= 64 ? launch_main<64>(A, static_cast<unsigned>(grid), st) : launch_main<128>(A, static_cast<unsigned>(grid), st);
}

}  // extern "C"
