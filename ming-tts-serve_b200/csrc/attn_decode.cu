// attn_decode.cu — attention of one new token per sequence over a paged cache,
// split over the cache's length and joined inside a thread-block cluster.
#include <cuda_runtime.h>

#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>

#include "attn.cuh"

namespace ming {

namespace {
namespace cg = cooperative_groups;

constexpr int DE_MAX_SPLIT = 16;          // CTAs of a cluster
constexpr int DE_OLD = AT_HD + 4;         // row of merged outputs: float4-aligned, rows on other banks
constexpr int de_part(int warps) { return warps * AT_MAXG * (DE_OLD + 2); }  // floats: every warp's outputs, maxima and sums
constexpr int de_smem(int warps) { return (de_part(warps) + AT_MAXG * (DE_OLD + 2) + 2 * AT_MAXG) * 4; }
constexpr int DE_SMEM_MAX = 200 * 1024;

enum { DE_PLAIN = 0, DE_TRACK = 1, DE_TRACK_AGAIN = 2 };

// The pages a row sees, counted 0 .. np - 1: the sinks' pages, then the
// window's. A page at an edge holds positions that are not seen.
struct SeenPages {
    int n, s1, w0, sp, wp, np;
    MING_DEV SeenPages(int len, int window, int sinks) {
        n = len;
        at_sees(n - 1, window, sinks, s1, w0);
        wp = w0 / AT_PAGE;
        sp = min((s1 + AT_PAGE - 1) / AT_PAGE, wp);
        np = n > 0 ? sp + (n + AT_PAGE - 1) / AT_PAGE - wp : 0;
    }
    MING_DEV int page(int i) const { return i < sp ? i : i - sp + wp; }
    MING_DEV bool sees(int j) const { return j < n && (j < s1 || j >= w0); }
    MING_DEV bool whole(int p) const { return p * AT_PAGE + AT_PAGE <= n && (p * AT_PAGE >= w0 || p * AT_PAGE + AT_PAGE <= s1); }
};

MING_DEV uint32_t de_prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }
}  // namespace

// A cluster per (sequence, kv head); its CTAs split the row's pages, a CTA's
// warps take them in turn. Per page of 16 positions a warp runs the group's
// heads (8 of the 16 rows of mma.sync m16n8k16; one token has too few rows for
// the 128-row tensor-memory instructions) against keys and values that come
// straight from global memory in the instructions' own fragment order:
//  * a sum over dims may run in any order, so lane (g, t) of a key fragment
//    takes bytes [16 t, 16 t + 16) and [64 + 16 t, ..) of position g's row,
//    two 16-byte loads, and q's fragments are permuted alike;
//  * output columns may carry any dim, so lane (g, t) of a value fragment
//    takes bytes [16 g, 16 g + 16) of rows 2t, 2t+1, 2t+8, 2t+9; column tile
//    i then holds dims 8 c + i of its columns c, and a lane ends up with 16
//    consecutive dims of one head.
// The next page's eight loads are issued before the current one's products:
// 4 KB in flight per warp, nothing staged in shared memory. Weights enter the
// second product as bf16 hi in rows 0-7 and lo in rows 8-15 (the rows that the
// group leaves empty), so they keep 16 bits at no cost. Softmax is one pass:
// running maximum and sum per warp, joined over warps, then over the cluster's
// CTAs through distributed shared memory; no workspace, no atomics, the order
// of sums fixed by the shapes.
// Tracking (the weights' running totals) needs the final maximum and sum:
// DE_TRACK keeps the logits in shared memory until the join, DE_TRACK_AGAIN
// (longer than fits) reads the keys a second time.
// Bound by: the cache's bytes (256 per position and kv head) for batches, the
// launch, two dependent loads and the cluster's two barriers for short rows.
// Measured (14 query, 2 kv heads): 64 x 4096 positions 28.6 us, 4.7 TB/s, and
// 38.0 us with tracking (its logits take the L1's room from the loads in
// flight); 1 x 509 5.0 us; 1 x 32768 16.0 us: a cluster sits in one part of
// the chip, whose share of the memory's rate is an eighth, so two heads alone
// cannot have all of it. Rings of cp.async three pages ahead and operands
// swapped for half the products changed none of this (34, 42 and 18 us).
template <int MODE, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, 16 / WARPS) attn_decode_kernel(const AttnOp a, int sc_ld) {
    constexpr int THREADS = WARPS * 32;
    extern __shared__ __align__(16) float de_buf[];
    float* wo = de_buf;                                  // [warp][head][DE_OLD]
    float* wm = wo + WARPS * AT_MAXG * DE_OLD;        // [warp][head]
    float* wl = wm + WARPS * AT_MAXG;
    float* co = de_buf + de_part(WARPS);                       // this CTA's [head][DE_OLD], unnormalised
    float* cm = co + AT_MAXG * DE_OLD;
    float* cl = cm + AT_MAXG;
    float* fm = cl + AT_MAXG;                            // the cluster's maxima and 1 / sums
    float* fl = fm + AT_MAXG;
    float* sc = fl + AT_MAXG;                            // DE_TRACK: logits [head][sc_ld]
    const int rank = blockIdx.x, ns = gridDim.x, kh = blockIdx.y, b = blockIdx.z;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int seq = at_seq(a.kv, b);
    const int* bt = a.kv.bt + (size_t)seq * a.kv.bt_ld;
    const SeenPages see(at_len_of(a.kv, seq, a.err), a.window, a.sinks);
    const int v0 = (int)((long long)see.np * rank / ns), v1 = (int)((long long)see.np * (rank + 1) / ns);

    // q fragments: row g, dims 8 t + 2 ks.. and 32 + 8 t + 2 ks..
    uint32_t qa[4][2];
    {
        const uint16_t* qr = a.q + b * a.q_rs + (kh * a.group + (g < a.group ? g : 0)) * a.q_hs;
        const uint4 x = reinterpret_cast<const uint4*>(qr)[t], y = reinterpret_cast<const uint4*>(qr)[t + 4];
        const bool has = g < a.group;
        qa[0][0] = has ? x.x : 0u, qa[1][0] = has ? x.y : 0u, qa[2][0] = has ? x.z : 0u, qa[3][0] = has ? x.w : 0u;
        qa[0][1] = has ? y.x : 0u, qa[1][1] = has ? y.y : 0u, qa[2][1] = has ? y.z : 0u, qa[3][1] = has ? y.w : 0u;
    }
    float m = -INFINITY, l = 0.f, o[8][4];
#pragma unroll
    for (int i = 0; i < 8; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;

    // this warp's pages: v0 + warp, + 8, ..; a lane looks up every 32nd ahead of use
    const int first = v0 + warp, count = first < v1 ? (v1 - first + WARPS - 1) / WARPS : 0;
    int ids = 0;
    auto look_up = [&](int i0) {
        const int i = i0 + lane;
        ids = i < count ? at_page(a.kv, bt, see.page(first + i * WARPS), a.err) : 0;
    };
    uint4 kf[4], vf[4];  // the page in flight
    auto fetch_k = [&](int64_t base) {
        const uint16_t* r0 = a.kv.k + base + g * a.kv.ss + 8 * t;
        const uint16_t* r8 = r0 + 8 * a.kv.ss;
        kf[0] = ldg_nc16(r0);
        kf[1] = ldg_nc16(r0 + 32);
        kf[2] = ldg_nc16(r8);
        kf[3] = ldg_nc16(r8 + 32);
    };
    auto fetch_v = [&](int64_t base) {
        const uint16_t* r0 = a.kv.v + base + 2 * t * a.kv.ss + 8 * g;
        vf[0] = ldg_nc16(r0);
        vf[1] = ldg_nc16(r0 + a.kv.ss);
        vf[2] = ldg_nc16(r0 + 8 * a.kv.ss);
        vf[3] = ldg_nc16(r0 + 9 * a.kv.ss);
    };
    auto base_of = [&](int i) { return (int64_t)__shfl_sync(0xffffffffu, ids, i & 31) * a.kv.ps + kh * a.kv.hs; };
    // logits of the page in kf: c[0..1] positions 2t, 2t+1, c[2..3] positions 8 + 2t, ..
    auto logits = [&](const uint4 (&k)[4], int p, float (&c)[4]) {
        float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
        const uint32_t kw[4][4] = {{k[0].x, k[1].x, k[2].x, k[3].x}, {k[0].y, k[1].y, k[2].y, k[3].y},
                                   {k[0].z, k[1].z, k[2].z, k[3].z}, {k[0].w, k[1].w, k[2].w, k[3].w}};
#pragma unroll
        for (int ks = 0; ks < 4; ks++) {
            const uint32_t q4[4] = {qa[ks][0], 0u, qa[ks][1], 0u};
            mma_bf16(x, q4, kw[ks][0], kw[ks][1]);
            mma_bf16(y, q4, kw[ks][2], kw[ks][3]);
        }
        c[0] = x[0] * a.scale_log2, c[1] = x[1] * a.scale_log2, c[2] = y[0] * a.scale_log2, c[3] = y[1] * a.scale_log2;
        if (!see.whole(p)) {
            const int j = p * AT_PAGE + 2 * t;
            if (!see.sees(j)) c[0] = -INFINITY;
            if (!see.sees(j + 1)) c[1] = -INFINITY;
            if (!see.sees(j + 8)) c[2] = -INFINITY;
            if (!see.sees(j + 9)) c[3] = -INFINITY;
        }
    };

    look_up(0);
    if (count > 0) {
        const int64_t base = base_of(0);
        fetch_k(base);
        fetch_v(base);
    }
    for (int i = 0; i < count; i++) {
        const int vi = first + i * WARPS, p = see.page(vi);
        uint4 k[4] = {kf[0], kf[1], kf[2], kf[3]}, v[4] = {vf[0], vf[1], vf[2], vf[3]};
        if (i + 1 < count) {
            if (((i + 1) & 31) == 0) look_up(i + 1);
            const int64_t base = base_of(i + 1);
            fetch_k(base);
            fetch_v(base);
        }
        float c[4];
        logits(k, p, c);
        if (MODE == DE_TRACK) {
            float* s = sc + g * sc_ld + (vi - v0) * AT_PAGE + 2 * t;
            *reinterpret_cast<float2*>(s) = make_float2(c[0], c[1]);
            *reinterpret_cast<float2*>(s + 8) = make_float2(c[2], c[3]);
        }
        if (!see.whole(p)) {  // 0 x NaN is NaN: values that are not seen become zeros
            const int j = p * AT_PAGE + 2 * t;
            if (!see.sees(j)) v[0] = make_uint4(0, 0, 0, 0);
            if (!see.sees(j + 1)) v[1] = make_uint4(0, 0, 0, 0);
            if (!see.sees(j + 8)) v[2] = make_uint4(0, 0, 0, 0);
            if (!see.sees(j + 9)) v[3] = make_uint4(0, 0, 0, 0);
        }
        float mx = fmaxf(fmaxf(c[0], c[1]), fmaxf(c[2], c[3]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        if (__any_sync(0xffffffffu, mx > m)) {
            const float mn = fmaxf(m, mx), r = exp2f(m - mn);
            m = mn;
            l *= r;
#pragma unroll
            for (int d = 0; d < 8; d++) o[d][0] *= r, o[d][1] *= r, o[d][2] *= r, o[d][3] *= r;
        }
        float e[4];
#pragma unroll
        for (int d = 0; d < 4; d++) e[d] = exp2f(c[d] - m);
        l += (e[0] + e[1]) + (e[2] + e[3]);
        const uint32_t h0 = at_bf16x2(e[0], e[1]), h1 = at_bf16x2(e[2], e[3]);
        const float2 f0 = unpack_bf16x2(h0), f1 = unpack_bf16x2(h1);
        const uint32_t pa[4] = {h0, at_bf16x2(e[0] - f0.x, e[1] - f0.y), h1, at_bf16x2(e[2] - f1.x, e[3] - f1.y)};
        const uint32_t vw[4][4] = {{v[0].x, v[1].x, v[2].x, v[3].x}, {v[0].y, v[1].y, v[2].y, v[3].y},
                                   {v[0].z, v[1].z, v[2].z, v[3].z}, {v[0].w, v[1].w, v[2].w, v[3].w}};
#pragma unroll
        for (int d = 0; d < 4; d++) {
            mma_bf16(o[2 * d], pa, de_prmt(vw[d][0], vw[d][1], 0x5410), de_prmt(vw[d][2], vw[d][3], 0x5410));
            mma_bf16(o[2 * d + 1], pa, de_prmt(vw[d][0], vw[d][1], 0x7632), de_prmt(vw[d][2], vw[d][3], 0x7632));
        }
    }
    // the warp's part: lane (g, t) holds dims 16 t .. 16 t + 15 of head g
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    if (t == 0) {
        wm[warp * AT_MAXG + g] = m;
        wl[warp * AT_MAXG + g] = l;
    }
    {
        float* w = wo + (warp * AT_MAXG + g) * DE_OLD + 16 * t;
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
            for (int d = 0; d < 8; d += 4)
                *reinterpret_cast<float4*>(w + 8 * c + d) = make_float4(o[d][c] + o[d][c + 2], o[d + 1][c] + o[d + 1][c + 2],
                                                                        o[d + 2][c] + o[d + 2][c + 2], o[d + 3][c] + o[d + 3][c + 2]);
    }
    __syncthreads();
    // the CTA's part: eight warps a head each, or sixteen half a head
    {
        constexpr int DIMS = 16 / WARPS;  // a lane's
        const int h = warp % AT_MAXG, d0 = (warp / AT_MAXG) * 32 + DIMS * lane;
        float M = -INFINITY, L = 0.f, x[DIMS] = {};
#pragma unroll
        for (int w = 0; w < WARPS; w++) M = fmaxf(M, wm[w * AT_MAXG + h]);
#pragma unroll
        for (int w = 0; w < WARPS; w++) {
            const float f = M == -INFINITY ? 0.f : exp2f(wm[w * AT_MAXG + h] - M);
            L += wl[w * AT_MAXG + h] * f;
#pragma unroll
            for (int d = 0; d < DIMS; d++) x[d] += wo[(w * AT_MAXG + h) * DE_OLD + d0 + d] * f;
        }
#pragma unroll
        for (int d = 0; d < DIMS; d++) co[h * DE_OLD + d0 + d] = x[d];
        if (lane == 0 && warp < AT_MAXG) cm[h] = M, cl[h] = L;
    }
    // the totals that this thread adds to, on their way while the parts meet
    float* const acc = MODE == DE_TRACK ? a.acc + seq * a.a_ss + kh * a.a_hs : nullptr;
    const int mine = (v1 - v0) * AT_PAGE;
    float old[4];
    auto position = [&](int e) { return see.page(v0 + e / AT_PAGE) * AT_PAGE + e % AT_PAGE; };
    auto fetch_acc = [&](int e0) {
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int e = e0 + k * THREADS, j = e < mine ? position(e) : see.n;
            old[k] = see.sees(j) && j != see.n - 1 ? acc[j] : 0.f;
        }
    };
    if (MODE == DE_TRACK) fetch_acc(tid);
    cg::cluster_group cluster = cg::this_cluster();
    if (ns > 1) cluster.sync();
    else __syncthreads();
    // the cluster's: the group's outputs, two dims at a time, over the ranks
    for (int e = rank * THREADS + tid; e < a.group * (AT_HD / 2); e += ns * THREADS) {
        const int h = e / (AT_HD / 2), d = e % (AT_HD / 2);
        float M = -INFINITY, L = 0.f, x = 0.f, y = 0.f;
        for (int r = 0; r < ns; r++) M = fmaxf(M, ns > 1 ? *cluster.map_shared_rank(cm + h, r) : cm[h]);
        for (int r = 0; r < ns; r++) {
            const float* po = ns > 1 ? cluster.map_shared_rank(co, r) : co;
            const float f = M == -INFINITY ? 0.f : exp2f(po[AT_MAXG * DE_OLD + h] - M);
            const float2 v = *reinterpret_cast<const float2*>(po + h * DE_OLD + 2 * d);
            L += po[AT_MAXG * DE_OLD + AT_MAXG + h] * f;
            x += v.x * f;
            y += v.y * f;
        }
        const float il = L > 0.f ? 1.f / L : 0.f;
        reinterpret_cast<uint32_t*>(a.out + b * a.o_rs + (kh * a.group + h) * a.o_hs)[d] = at_bf16x2(x * il, y * il);
    }
    if (MODE != DE_PLAIN) {
        if (tid < AT_MAXG) {
            float M = -INFINITY, L = 0.f;
            for (int r = 0; r < ns; r++) M = fmaxf(M, ns > 1 ? *cluster.map_shared_rank(cm + tid, r) : cm[tid]);
            for (int r = 0; r < ns; r++) {
                const float* pm = ns > 1 ? cluster.map_shared_rank(cm, r) : cm;
                L += M == -INFINITY ? 0.f : pm[AT_MAXG + tid] * exp2f(pm[tid] - M);
            }
            fm[tid] = M;
            fl[tid] = L > 0.f ? 1.f / L : 0.f;
        }
        __syncthreads();
        if (MODE == DE_TRACK) {
            for (int e0 = tid; e0 < mine; e0 += 4 * THREADS) {
                float now[4];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const int e = e0 + k * THREADS;
                    float w = 0.f;
                    if (e < mine)
                        for (int h = 0; h < a.group; h++) w += exp2f(sc[h * sc_ld + e] - fm[h]) * fl[h];
                    now[k] = old[k] + w;
                }
                fetch_acc(e0 + 4 * THREADS);
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const int e = e0 + k * THREADS, j = e < mine ? position(e) : see.n;
                    if (see.sees(j)) acc[j] = now[k];
                }
            }
        } else {
            const float M = fm[g], il = g < a.group ? fl[g] : 0.f;
            look_up(0);
            for (int i = 0; i < count; i++) {
                if (i > 0 && (i & 31) == 0) look_up(i);
                const int p = see.page(first + i * WARPS);
                fetch_k(base_of(i));
                float c[4];
                logits(kf, p, c);
#pragma unroll
                for (int d = 0; d < 4; d++) {
                    float w = g < a.group ? exp2f(c[d] - M) * il : 0.f;
#pragma unroll
                    for (int s = 4; s < 32; s <<= 1) w += __shfl_xor_sync(0xffffffffu, w, s);
                    const int j = p * AT_PAGE + 2 * t + (d & 1) + 4 * (d & 2);
                    float* total = a.acc + seq * a.a_ss + kh * a.a_hs + j;
                    if (g == 0 && see.sees(j)) *total = (j == see.n - 1 ? 0.f : *total) + w;
                }
            }
        }
    }
    if (ns > 1) cluster.sync();  // the others may still be reading this CTA's part
}

cudaError_t launch_attn_decode(const AttnOp& a, cudaStream_t s) {
    static std::atomic<bool> ready[64] = {};  // per device: the kernels' attributes are set
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !ready[dev].load(std::memory_order_acquire)) {
        const void* f[6] = {(const void*)attn_decode_kernel<DE_PLAIN, 8>,       (const void*)attn_decode_kernel<DE_TRACK, 8>,
                            (const void*)attn_decode_kernel<DE_TRACK_AGAIN, 8>, (const void*)attn_decode_kernel<DE_PLAIN, 16>,
                            (const void*)attn_decode_kernel<DE_TRACK, 16>,      (const void*)attn_decode_kernel<DE_TRACK_AGAIN, 16>};
        for (const void* k : f) {
            if ((e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, DE_SMEM_MAX)) != cudaSuccess) return e;
            if ((e = cudaFuncSetAttribute(k, cudaFuncAttributeNonPortableClusterSizeAllowed, 1)) != cudaSuccess) return e;
        }
        if (dev < 64) ready[dev].store(true, std::memory_order_release);
    }
    // pages a row can see at most (both edges of the window may be in the middle of one)
    const long long most = ((long long)a.kv.max_len + AT_PAGE - 1) / AT_PAGE;
    const long long pages =
        a.window ? std::min(most, ((long long)a.window + 2 * AT_PAGE - 2) / AT_PAGE +
                                      std::min(most, ((long long)a.sinks + AT_PAGE - 1) / AT_PAGE))
                 : most;
    // Splits: as many as fill the SMs once, two CTAs each, if there are pages
    // enough to give each warp one. (64 x 4096 positions, 128 heads: 42 us in
    // one part, 29 in two, 34 in four, 46 in eight.) Clusters of sixteen find
    // place one at a time in each part of the chip: for few heads alone (8 x
    // 4096, 16 heads: 10.4 us in eight parts, 16.5 in sixteen; 1 x 4096: 8.6
    // and 7.6). Sixteen warps a CTA pay on a cache that gives each warp four
    // pages (1 x 32768: 15.8 us against 18.9; 1 x 2048: 7.3 against 6.5).
    const long long heads = (long long)a.seqs * a.kv_heads;
    int ns = 1;
    while (ns < DE_MAX_SPLIT && heads * ns * 2 <= (ns == 8 ? 64 : 2 * 148) && pages >= 2 * ns * 8) ns *= 2;
    const int warps = heads * ns <= 64 && pages >= 4 * 16 * ns ? 16 : 8;
    auto ld_of = [&](int ns) {  // 8 past a multiple of 32: the eight heads' stores fall on distinct banks
        return (pages + ns - 1) / ns * AT_PAGE / 32 * 32 + 40;
    };
    auto track = [&](int ns) { return de_smem(warps) + ld_of(ns) * AT_MAXG * 4; };
    int mode = DE_PLAIN, ld = 0;
    size_t smem = de_smem(warps);
    if (a.acc) {
        // logits leave the L1 room for the loads in flight: with 86 KB of them
        // a CTA (two parts) 64 x 4096 positions took 41.5 us, with 53 KB 38.4
        while (ns < 8 && heads * ns > 148 && track(ns) > 56 * 1024) ns *= 2;
        mode = track(ns) <= DE_SMEM_MAX ? DE_TRACK : DE_TRACK_AGAIN;
        if (mode == DE_TRACK) {
            smem = track(ns);
            ld = (int)ld_of(ns);
        }
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ns, a.kv_heads, a.seqs);
    cfg.blockDim = dim3(warps * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = ns;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    using Kernel = void (*)(AttnOp, int);
    static const Kernel kernels[2][3] = {
        {attn_decode_kernel<DE_PLAIN, 8>, attn_decode_kernel<DE_TRACK, 8>, attn_decode_kernel<DE_TRACK_AGAIN, 8>},
        {attn_decode_kernel<DE_PLAIN, 16>, attn_decode_kernel<DE_TRACK, 16>, attn_decode_kernel<DE_TRACK_AGAIN, 16>}};
    return cudaLaunchKernelEx(&cfg, kernels[warps == 16][mode], a, ld);
}

}  // namespace ming
