// attn_prefill.cu — attention of a prompt's rows over a paged cache, and the
// weights that those rows gave to each cached position, on the 5th-generation
// tensor cores (tcgen05.mma, sums in tensor memory).
#include <cuda_runtime.h>

#include <atomic>

#include "attn.cuh"

namespace ming {

namespace {

constexpr int PF_M = 128;        // rows of a tile: (position, head of the group) pairs
constexpr int PF_N = 128;        // cached positions of a block: eight pages
constexpr int PF_PAGES = PF_N / AT_PAGE;
constexpr int PF_STAGES = 4;
constexpr int PF_TILE = PF_M * AT_HD * 2;  // 16 KB: a row of 64 bf16 is one 128-byte swizzled line
constexpr int PF_THREADS = 384;            // two softmax warpgroups, then one MMA warp and three loading warps
constexpr int PF_LOADERS = 96;
constexpr int PF_SMEM = 1024 + 2 * PF_TILE + PF_STAGES * 2 * PF_TILE + 256;
constexpr long long PF_TIMEOUT = 4000000000LL;  // cycles (~2 s) before a wait gives up; the ones here end in microseconds
// tensor memory columns
constexpr int PF_S = 0;    // logits of the two tiles, f32 [128 rows][128]
constexpr int PF_P = 256;  // weights of the two tiles, bf16 pairs [128 rows][64]
constexpr int PF_O = 384;  // outputs of the two tiles, f32 [128 rows][64]
constexpr int PF_COLS = 512;

MING_DEV uint32_t pf_su32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
MING_DEV void pf_bar_init(uint64_t* b, int count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(pf_su32(b)), "r"(count) : "memory");
}
MING_DEV void pf_arrive(uint64_t* b) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(pf_su32(b)) : "memory");
}
MING_DEV bool pf_try(uint64_t* b, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(pf_su32(b)), "r"(parity)
        : "memory");
    return ok != 0;
}
MING_DEV bool pf_wait(uint64_t* b, uint32_t parity) {
    if (pf_try(b, parity)) return true;
    const long long t0 = clock64();
    while (!pf_try(b, parity))
        if (clock64() - t0 > PF_TIMEOUT) return false;
    return true;
}
// The whole warp waits and agrees on the outcome.
MING_DEV bool pf_wait_warp(uint64_t* b, uint32_t parity) { return __all_sync(0xffffffffu, pf_wait(b, parity)); }
MING_DEV void pf_commit(uint64_t* b) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(pf_su32(b)) : "memory");
}
MING_DEV void pf_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
MING_DEV void pf_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
MING_DEV void pf_async_fence() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }

// Shared-memory matrix descriptor of a tile of 128-byte rows, 128-byte swizzle,
// groups of eight rows 1024 bytes apart: as [rows][64 K] (K-major) and, with
// the instruction's transpose bit, as [K rows][64 columns] alike.
MING_DEV uint64_t pf_desc(uint32_t saddr) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) |
           ((uint64_t)2 << 61);
}
// Instruction descriptors (kind::f16): f32 sums, bf16 operands, M 128; B
// K-major of N 128 for q.k, B transposed of N 64 for the weights' product.
constexpr uint32_t PF_IDESC = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(PF_M >> 4) << 24);
constexpr uint32_t PF_IDESC_QK = PF_IDESC | ((uint32_t)(PF_N >> 3) << 17);
constexpr uint32_t PF_IDESC_PV = PF_IDESC | ((uint32_t)(AT_HD >> 3) << 17) | (1u << 16);

MING_DEV void pf_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
        : "memory");
}
MING_DEV void pf_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
        : "memory");
}
// A 128 x 128 x 64 product of two K-major tiles
MING_DEV void pf_product(uint32_t d, uint32_t a, uint32_t b) {
#pragma unroll
    for (int ks = 0; ks < 4; ks++) pf_mma_ss(d, pf_desc(a + 32 * ks), pf_desc(b + 32 * ks), PF_IDESC_QK, ks > 0);
}

#define PF_R8(v, i) "=r"((v)[i]), "=r"((v)[i + 1]), "=r"((v)[i + 2]), "=r"((v)[i + 3]), "=r"((v)[i + 4]), "=r"((v)[i + 5]), "=r"((v)[i + 6]), "=r"((v)[i + 7])
#define PF_W8(v, i) "r"((v)[i]), "r"((v)[i + 1]), "r"((v)[i + 2]), "r"((v)[i + 3]), "r"((v)[i + 4]), "r"((v)[i + 5]), "r"((v)[i + 6]), "r"((v)[i + 7])
// 32 columns of the warp's 32 lanes
MING_DEV void pf_ld32(uint32_t* v, uint32_t addr) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
        : PF_R8(v, 0), PF_R8(v, 8), PF_R8(v, 16), PF_R8(v, 24)
        : "r"(addr));
}
MING_DEV void pf_st32(uint32_t addr, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};\n" ::"r"(
            addr),
        PF_W8(v, 0), PF_W8(v, 8), PF_W8(v, 16), PF_W8(v, 24)
        : "memory");
}
// Waits for the loads into v; the empty statements keep its uses behind the wait.
template <int N>
MING_DEV void pf_wait_ld(uint32_t (&v)[N]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; i++) asm volatile("" : "+r"(v[i]));
}
MING_DEV void pf_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }

MING_DEV float pf_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
// Two f32 operations in one instruction
MING_DEV uint64_t pf_pair(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
MING_DEV void pf_unpair(uint64_t r, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;\n" : "=f"(x), "=f"(y) : "l"(r)); }
MING_DEV uint64_t pf_fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
MING_DEV uint64_t pf_add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// bits [a, b) of a word
MING_DEV uint32_t pf_bits(int a, int b) {
    a = max(a, 0);
    b = min(b, 32);
    return b <= a ? 0u : (0xffffffffu >> (32 - b)) & (0xffffffffu << a);
}

// The pages that the rows at positions [pa, pb] of a sequence see between
// them, counted 0 .. np - 1: the sinks' pages, then the window's. Blocks are
// PF_PAGES of them.
struct RowsSee {
    int pb, w0, window, sinks, sp, wp, np;
    MING_DEV RowsSee(int pa, int pb_, int window_, int sinks_) : pb(pb_), window(window_), sinks(sinks_) {
        int s1;
        at_sees(pa, window, sinks, s1, w0);
        wp = w0 / AT_PAGE;
        sp = min((s1 + AT_PAGE - 1) / AT_PAGE, wp);
        np = pb >= 0 ? sp + pb / AT_PAGE + 1 - wp : 0;
    }
    MING_DEV int page(int i) const { return i < sp ? i : i - sp + wp; }
    MING_DEV int blocks() const { return (np + PF_PAGES - 1) / PF_PAGES; }
    MING_DEV bool any(int j) const { return j <= pb && (j < sinks || j >= w0); }
    MING_DEV bool all(int page) const {
        const int j = page * AT_PAGE;
        return j + AT_PAGE - 1 <= pb && (j >= w0 || j + AT_PAGE <= sinks);
    }
};

// Which columns of a block a row sees: columns [0, cs) are positions ja + c of
// the sinks' pages, columns [cs, 128) positions jb + c.
struct BlockSpan {
    int cs, ja, jb;
    MING_DEV BlockSpan(const RowsSee& r, int block) {
        const int v0 = block * PF_PAGES;
        cs = min(max((r.sp - v0) * AT_PAGE, 0), PF_N);
        ja = v0 * AT_PAGE;
        jb = (v0 - r.sp + r.wp) * AT_PAGE;
    }
    // every row at positions [pa, pb] sees every column
    MING_DEV bool whole(int pa, int pb, int window, int sinks) const {
        if (cs == PF_N) return ja + PF_N <= sinks;
        return cs == 0 && jb + PF_N - 1 <= pa && (!window || jb > pb - window || jb + PF_N <= sinks);
    }
    MING_DEV uint32_t sees(int c0, int p, int window, int sinks) const {
        const int end = p - jb + 1, lo = window ? p - window + 1 - jb : 0;
        return pf_bits(-c0, min(cs, min(sinks, p + 1) - ja) - c0) | pf_bits(cs - c0, min(sinks - jb, end) - c0) |
               pf_bits(max(cs, lo) - c0, end - c0);
    }
};

// The loading warps copy one block's keys and values into swizzled tiles, a
// warp a page at a time, 16 bytes a lane; rows that no row of the CTA sees
// become zeros (a weight of zero times a stale NaN would be NaN).
MING_DEV void pf_load_block(const KvPages& kv, const int* bt, const RowsSee& see, int kh, int block, uint8_t* tiles, int lw,
                            int lane, bool values, int* err) {
    const int v = block * PF_PAGES + (lane & 7);
    const int mine = v < see.np ? see.page(v) : -1;
    const int64_t base = mine >= 0 ? (int64_t)at_page(kv, bt, mine, err) * kv.ps + kh * kv.hs : 0;
    const int row = lane >> 3, chunk = lane & 7;
    const int64_t off = row * kv.ss + chunk * 8, step = 4 * kv.ss;
    const uint32_t at = pf_su32(tiles) + row * 128;
    const uint32_t c0 = (uint32_t)(chunk ^ row) << 4, c1 = (uint32_t)(chunk ^ (row + 4)) << 4;
    for (int u = lw; u < (values ? 2 : 1) * PF_PAGES; u += PF_LOADERS / 32) {
        const int pi = u & (PF_PAGES - 1);
        const int page = __shfl_sync(0xffffffffu, mine, pi);
        const uint16_t* s = (u < PF_PAGES ? kv.k : kv.v) + __shfl_sync(0xffffffffu, base, pi) + off;
        const uint32_t d = at + (u < PF_PAGES ? 0 : PF_TILE) + pi * (AT_PAGE * 128);
        const int j = page * AT_PAGE + row;
        const bool whole = page >= 0 && see.all(page);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const bool live = whole || (page >= 0 && see.any(j + 4 * k));
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(d + k * 512 + (k & 1 ? c1 : c0)), "l"(s + k * step),
                         "r"(live ? 16 : 0)
                         : "memory");
        }
    }
}

// One (position, head) row of q into line r of a swizzled tile, zeros if there is none.
MING_DEV void pf_load_q(const AttnOp& a, uint8_t* tile, int r, int64_t row, int h, bool has) {
    const uint4* s = reinterpret_cast<const uint4*>(a.q + row * a.q_rs + h * a.q_hs);
#pragma unroll
    for (int c = 0; c < 8; c++)
        *reinterpret_cast<uint4*>(tile + r * 128 + ((c ^ (r & 7)) << 4)) = has ? s[c] : make_uint4(0, 0, 0, 0);
}

}  // namespace

// A CTA takes two tiles of 128 rows of one (sequence, kv head): a row is a
// (position, head of the group) pair, so a block of keys and values serves the
// whole group and the tile's mask is as narrow as its 128 / group positions.
// Per block of 128 cached positions and tile: logits S = Q K^T into tensor
// memory (4 tcgen05.mma), a thread per row reads its 128 logits, keeps the
// running maximum and sum in registers, writes the weights as bf16 pairs back
// to tensor memory, and O += P V takes them from there (8 tcgen05.mma with V
// as the transposed operand, its rows as the pages hold them). Nothing of S or
// P passes through shared memory, and no row needs a shuffle.
//  * Outputs are rescaled only when a row's maximum has risen by more than 2^8
//    since the last time (sums and outputs carry the same reference, so the
//    quotient is exact; weights stay below 2^8).
//  * P is rounded to bf16, half a step of each weight, because the tensor
//    cores take bf16 next to V; the row's sum is kept from the unrounded ones.
//  * Softmax of one tile runs while the other's products do; q.k of the next
//    block is issued as soon as a tile's logits have been read.
//  * Three warps bring blocks in with 16-byte cp.async (pages may sit at any
//    stride), four stages of 32 KB ahead.
__global__ void __launch_bounds__(PF_THREADS, 1) attn_prefill_kernel(const AttnOp a) {
    extern __shared__ __align__(16) uint8_t pf_raw[];
    uint8_t* smem = pf_raw + ((1024u - (pf_su32(pf_raw) & 1023u)) & 1023u);
    uint8_t* sq = smem;                    // [2] tiles of q
    uint8_t* skv = smem + 2 * PF_TILE;     // [stage][K|V]
    uint64_t* bars = reinterpret_cast<uint64_t*>(skv + PF_STAGES * 2 * PF_TILE);
    uint64_t *full = bars, *empty = bars + PF_STAGES, *s_full = bars + 2 * PF_STAGES, *s_read = s_full + 2,
             *p_ready = s_full + 4, *o_full = s_full + 6;
    uint32_t* slot = reinterpret_cast<uint32_t*>(s_full + 8);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int kh = blockIdx.y, b = blockIdx.z, G = a.group, per = PF_M / G;  // positions of a tile
    int r0, r1;
    at_rows(a, b, r0, r1);
    const int rows = r1 - r0, x = gridDim.x - 1 - blockIdx.x, i0 = x * 2 * per;  // the longest rows first
    if (i0 >= rows) return;
    const int seq = at_seq(a.kv, b), len = at_len(a.kv, seq, a.err), p0 = len - rows + i0;
    const int* bt = a.kv.bt + (size_t)seq * a.kv.bt_ld;
    const int here = min(rows - i0, 2 * per), tiles = here > per ? 2 : 1;
    const RowsSee see(max(p0, 0), p0 + here - 1, a.window, a.sinks);
    const int nb = see.blocks();

    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(pf_su32(slot)), "r"(PF_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    if (tid == 0) {
        for (int i = 0; i < PF_STAGES; i++) {
            pf_bar_init(&full[i], PF_LOADERS);
            pf_bar_init(&empty[i], 1);
        }
        for (int t = 0; t < 2; t++) {
            pf_bar_init(&s_full[t], 1);
            pf_bar_init(&s_read[t], 4);
            pf_bar_init(&p_ready[t], 4);
            pf_bar_init(&o_full[t], 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    const int t = warp >> 2;                       // softmax warps: the tile
    const int r = tid & 127, i = i0 + t * per + r / G, h = kh * G + r % G;
    const bool has = t < 2 && r < per * G && i < rows;
    if (t < 2) {
        pf_load_q(a, sq + t * PF_TILE, r, r0 + i, h, has);
        pf_async_fence();
    }
    pf_before();
    __syncthreads();
    pf_after();
    const uint32_t tmem = *slot;
    bool ok = true;
    if (warp == 8) {
        if (lane == 0 && nb > 0) {
            auto kv_at = [&](int j) { return pf_su32(skv) + (uint32_t)(j % PF_STAGES) * 2 * PF_TILE; };
            ok = pf_wait(&full[0], 0);
            for (int u = 0; ok && u < tiles; u++) {
                pf_product(tmem + PF_S + u * PF_N, pf_su32(sq) + u * PF_TILE, kv_at(0));
                pf_commit(&s_full[u]);
            }
            for (int j = 0; ok && j < nb; j++) {
                for (int u = 0; ok && u < tiles; u++) {
                    if (j + 1 < nb) {
                        if (u == 0) ok = pf_wait(&full[(j + 1) % PF_STAGES], ((j + 1) / PF_STAGES) & 1);
                        ok = ok && pf_wait(&s_read[u], j & 1);
                        if (!ok) break;
                        pf_after();
                        pf_product(tmem + PF_S + u * PF_N, pf_su32(sq) + u * PF_TILE, kv_at(j + 1));
                        pf_commit(&s_full[u]);
                    }
                    if (!(ok = pf_wait(&p_ready[u], j & 1))) break;
                    pf_after();
#pragma unroll
                    for (int ks = 0; ks < PF_N / 16; ks++)
                        pf_mma_ts(tmem + PF_O + u * AT_HD, tmem + PF_P + u * (PF_N / 2) + ks * 8,
                                  pf_desc(kv_at(j) + PF_TILE + ks * 2048), PF_IDESC_PV, j > 0 || ks > 0);
                    pf_commit(&o_full[u]);
                }
                if (ok) pf_commit(&empty[j % PF_STAGES]);
            }
        }
        __syncwarp();
    } else if (warp > 8) {
        const int lw = warp - 9;
        for (int j = 0; ok && j <= nb; j++) {
            if (j < nb) {
                if (j >= PF_STAGES) ok = pf_wait_warp(&empty[j % PF_STAGES], ((j / PF_STAGES) - 1) & 1);
                if (ok) {
                    uint8_t* st = skv + (j % PF_STAGES) * 2 * PF_TILE;
                    pf_load_block(a.kv, bt, see, kh, j, st, lw, lane, true, a.err);
                }
            }
            asm volatile("cp.async.commit_group;\n" ::: "memory");
            if (j > 0) {
                // the block before this one is in: hand it over
                asm volatile("cp.async.wait_group 1;\n" ::: "memory");
                pf_async_fence();
                pf_arrive(&full[(j - 1) % PF_STAGES]);
            }
        }
        asm volatile("cp.async.wait_group 0;\n" ::: "memory");
    } else if (t < tiles) {
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + lanes + PF_S + t * PF_N, tp = tmem + lanes + PF_P + t * (PF_N / 2),
                       to = tmem + lanes + PF_O + t * AT_HD;
        const int p = has ? p0 + t * per + r / G : -1;
        const int pa = p0 + t * per, pb = p0 + min(here, (t + 1) * per) - 1;
        float m = -INFINITY, l = 0.f;  // reference maximum (of q.k) and sum of the weights against it
        for (int j = 0; j < nb; j++) {
            if (!(ok = pf_wait_warp(&s_full[t], j & 1))) break;
            pf_after();
            uint32_t s[PF_N];
#pragma unroll
            for (int c = 0; c < PF_N; c += 32) pf_ld32(s + c, ts + c);
            pf_wait_ld(s);
            pf_before();
            __syncwarp();
            if (lane == 0) pf_arrive(&s_read[t]);
            const BlockSpan span(see, j);
            if (!span.whole(pa, pb, a.window, a.sinks)) {
#pragma unroll
                for (int c = 0; c < PF_N; c += 32) {
                    const uint32_t bits = span.sees(c, p, a.window, a.sinks);
#pragma unroll
                    for (int e = 0; e < 32; e++)
                        if (!((bits >> e) & 1u)) s[c + e] = 0xff800000u;  // -infinity
                }
            }
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < PF_N; c += 8)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    mx[e] = fmaxf(mx[e], fmaxf(__uint_as_float(s[c + 2 * e]), __uint_as_float(s[c + 2 * e + 1])));
            const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
            float f = 1.f;
            const bool rise = top > m && (top - m) * a.scale_log2 > 8.f;  // also from -infinity
            if (rise) {
                f = m == -INFINITY ? 0.f : pf_ex2((m - top) * a.scale_log2);
                m = top;
                l *= f;
            }
            const float ref = m == -INFINITY ? 0.f : -m * a.scale_log2;
            const uint64_t sc2 = pf_pair(a.scale_log2, a.scale_log2), ref2 = pf_pair(ref, ref);
            uint64_t sum[2] = {0ull, 0ull};
            uint32_t w[PF_N / 2];
#pragma unroll
            for (int c = 0; c < PF_N; c += 2) {
                float e0, e1;
                pf_unpair(pf_fma2(pf_pair(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), sc2, ref2), e0, e1);
                e0 = pf_ex2(e0);
                e1 = pf_ex2(e1);
                sum[(c >> 1) & 1] = pf_add2(sum[(c >> 1) & 1], pf_pair(e0, e1));
                w[c / 2] = at_bf16x2(e0, e1);
            }
            float u0, u1;
            pf_unpair(pf_add2(sum[0], sum[1]), u0, u1);
            l += u0 + u1;
            if (j > 0) {
                if (!(ok = pf_wait_warp(&o_full[t], (j - 1) & 1))) break;  // the last block's product has read P and written O
                pf_after();
                if (__any_sync(0xffffffffu, rise)) {
#pragma unroll
                    for (int c = 0; c < AT_HD; c += 32) {
                        uint32_t o[32];
                        pf_ld32(o, to + c);
                        pf_wait_ld(o);
#pragma unroll
                        for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                        pf_st32(to + c, o);
                    }
                }
            }
            pf_st32(tp, w);
            pf_st32(tp + 32, w + 32);
            pf_wait_st();
            pf_before();
            __syncwarp();
            if (lane == 0) pf_arrive(&p_ready[t]);
        }
        if (ok && nb > 0) ok = pf_wait_warp(&o_full[t], (nb - 1) & 1);
        pf_after();
        const float il = ok && l > 0.f ? 1.f / l : 0.f;
#pragma unroll
        for (int c = 0; c < AT_HD; c += 32) {
            uint32_t o[32];
            pf_ld32(o, to + c);
            pf_wait_ld(o);
            if (has) {
                uint4* d = reinterpret_cast<uint4*>(a.out + (int64_t)(r0 + i) * a.o_rs + h * a.o_hs + c);
#pragma unroll
                for (int e = 0; e < 32; e += 8) {
                    uint32_t y[4];
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        // nothing seen: zeros, whatever the tensor memory held
                        y[k] = l > 0.f || l != l ? at_bf16x2(__uint_as_float(o[e + 2 * k]) * il, __uint_as_float(o[e + 2 * k + 1]) * il) : 0u;
                    d[e / 8] = make_uint4(y[0], y[1], y[2], y[3]);
                }
            }
        }
        if (has && a.lse) a.lse[(size_t)(r0 + i) * a.heads + h] = l == 0.f ? -INFINITY : (m * a.scale_log2 + log2f(l)) / AT_LOG2E;
    }
    if (!ok) at_flag(a.err, AT_ERR_WAIT);
    pf_before();
    __syncthreads();
    if (warp == 8) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(PF_COLS) : "memory");
}

// One thread per cached position, its key in registers; the rows that see it
// follow one another.
__global__ void __launch_bounds__(128) attn_weights_kernel(const AttnOp a) {
    const int b = blockIdx.z, kh = blockIdx.y, j = blockIdx.x * 128 + threadIdx.x;
    int r0, r1;
    at_rows(a, b, r0, r1);
    const int seq = at_seq(a.kv, b), n = at_len(a.kv, seq, a.err), first = n - (r1 - r0);
    if (j >= n) return;
    const int* bt = a.kv.bt + (size_t)seq * a.kv.bt_ld;
    const uint16_t* kr =
        a.kv.k + (int64_t)at_page(a.kv, bt, j / AT_PAGE, a.err) * a.kv.ps + kh * a.kv.hs + (j % AT_PAGE) * a.kv.ss;
    float k[AT_HD];
    for (int d = 0; d < AT_HD; d++) k[d] = bf2f(kr[d]);
    float w = 0.f;
    for (int r = r0; r < r1; r++) {
        const int p = first + (r - r0);
        if (j > p || (a.window && j >= a.sinks && j <= p - a.window)) continue;
        for (int h = kh * a.group; h < (kh + 1) * a.group; h++) {
            const uint16_t* qr = a.q + r * a.q_rs + h * a.q_hs;
            float s = 0.f;
            for (int d = 0; d < AT_HD; d++) s += bf2f(qr[d]) * k[d];
            w += exp2f(s * a.scale_log2 - a.lse[(size_t)r * a.heads + h] * AT_LOG2E);
        }
    }
    float* t = a.acc + seq * a.a_ss + kh * a.a_hs + j;
    *t = (j >= first ? 0.f : *t) + w;
}

cudaError_t launch_attn_prefill(const AttnOp& a, cudaStream_t s) {
    static std::atomic<bool> ready[64] = {};  // per device: the kernel's attribute is set
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !ready[dev].load(std::memory_order_acquire)) {
        if ((e = cudaFuncSetAttribute(attn_prefill_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, PF_SMEM)) != cudaSuccess)
            return e;
        if (dev < 64) ready[dev].store(true, std::memory_order_release);
    }
    const int per = 2 * (PF_M / a.group);
    attn_prefill_kernel<<<dim3((a.max_rows + per - 1) / per, a.kv_heads, a.seqs), PF_THREADS, PF_SMEM, s>>>(a);
    return cudaGetLastError();
}

cudaError_t launch_attn_weights(const AttnOp& a, cudaStream_t s) {
    attn_weights_kernel<<<dim3((a.kv.max_len + 127) / 128, a.kv_heads, a.seqs), 128, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace ming
