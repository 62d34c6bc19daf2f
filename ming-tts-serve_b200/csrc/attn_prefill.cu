// attn_prefill.cu — attention of a prompt's rows over a paged cache, and the
// weights that those rows gave to each cached position, on the 5th-generation
// tensor cores (tcgen05.mma, sums in tensor memory).
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>

#include "attn.cuh"

namespace ming {

namespace {

constexpr int PF_M = 128;        // rows of a tile: (position, head of the group) pairs
constexpr int PF_N = 128;        // cached positions of a block: eight pages
constexpr int PF_PAGES = PF_N / AT_PAGE;
constexpr int PF_STAGES = 4;
constexpr int PF_TILE = PF_M * AT_HD * 2;  // 16 KB: a row of 64 bf16 is one 128-byte swizzled line
constexpr int PF_THREADS = 352;            // two softmax warpgroups, then a warp each for products, copies and edges
constexpr int PF_SMEM = 1024 + 4 * PF_TILE + PF_STAGES * 2 * PF_TILE + 2 * PF_TILE + 256;
constexpr long long PF_TIMEOUT = 4000000000LL;  // cycles (~2 s) before a wait gives up; the ones here end in microseconds
// tensor memory columns
constexpr int PF_BUFS = 3;  // logits of three (block, tile) steps, f32 [128 rows][128]; a step's weights replace its
                            // logits, bf16 pairs [128 rows][64]
constexpr int PF_O = 384;   // outputs of the two tiles, f32 [128 rows][64]
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
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(pf_su32(b)), "r"(parity), "r"(1000000)  // sleeps up to a millisecond instead of spinning beside warps at work
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
MING_DEV bool pf_elect() {
    uint32_t one;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.b32 %0, 1, 0, p;\n}\n" : "=r"(one));
    return one != 0;
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
MING_DEV uint64_t pf_desc_lo(uint32_t addr16) {  // of an address in units of 16 bytes
    return (uint64_t)(addr16 & 0x3FFFu) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
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
MING_DEV void pf_ld16(uint32_t* v, uint32_t addr) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
        : PF_R8(v, 0), PF_R8(v, 8)
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
MING_DEV void pf_st16(uint32_t addr, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n" ::"r"(addr),
        PF_W8(v, 0), PF_W8(v, 8)
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

MING_DEV void pf_expect(uint64_t* b, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(pf_su32(b)), "r"(bytes) : "memory");
}
// A page of one kv head: 16 rows of 128 bytes, swizzled. Page `pages` lies outside the map and gives zeros.
MING_DEV void pf_copy_page(void* dst, const CUtensorMap* m, int kh, int page, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %2, %3, %4}], [%5];\n" ::"r"(
            pf_su32(dst)),
        "l"(reinterpret_cast<uint64_t>(m)), "r"(0), "r"(kh), "r"(page), "r"(pf_su32(bar))
        : "memory");
}
// A tile of q: every head of the group at 128 / group positions from `row` on.
MING_DEV void pf_copy_q(void* dst, const CUtensorMap* m, int head, int row, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(
            pf_su32(dst)),
        "l"(reinterpret_cast<uint64_t>(m)), "r"(0), "r"(head), "r"(row), "r"(pf_su32(bar))
        : "memory");
}

// The work of a CTA, one (sequence, kv head, up to two tiles of rows) after
// another; the sequences' last rows, which see the most, come first.
struct PfItem {
    int kh, b, x;     // kv head, row of the batch, which rows
    int r0, r1, len;  // as read: rows of q, positions held
    MING_DEV PfItem() {}
    // The loads alone: their checks wait until the item's turn.
    MING_DEV void read(const AttnOp& a, int w, int nx) {
        const int per = a.kv_heads * a.seqs, rest = w % per;
        x = nx - 1 - w / per;
        b = rest / a.kv_heads;
        kh = rest % a.kv_heads;
        r0 = a.q_start[b];
        r1 = a.q_start[b + 1];
        len = a.kv.lens[at_seq(a.kv, b)];
    }
    MING_DEV void check(const AttnOp& a) {
        at_rows(a, r0, r1);
        len = at_len(a.kv, len + a.kv.len_add, a.err);
    }
};
// A CTA's items in turn, each read while the one before it is worked on.
struct PfItems {
    const AttnOp& a;
    int w, nx, total;
    PfItem ahead;
    MING_DEV PfItems(const AttnOp& a_, int nx_, int total_) : a(a_), w(blockIdx.x), nx(nx_), total(total_) {
        if (w < total) ahead.read(a, w, nx);
    }
    MING_DEV bool next(PfItem& it) {
        if (w >= total) return false;
        it = ahead;
        if ((w += gridDim.x) < total) ahead.read(a, w, nx);
        it.check(a);
        return true;
    }
};
struct PfRows {
    int i0, p0, here;  // first row within the sequence, its position, rows of the item (<= 0: none)
    MING_DEV PfRows(const PfItem& w, int step) {
        i0 = w.x * step;
        p0 = w.len - (w.r1 - w.r0) + i0;
        here = min(w.r1 - w.r0 - i0, step);
    }
    MING_DEV RowsSee see(const AttnOp& a) const { return RowsSee(max(p0, 0), p0 + here - 1, a.window, a.sinks); }
};

}  // namespace

// One CTA per SM takes items of two tiles of 128 rows of one (sequence, kv
// head): a row is a (position, head of the group) pair, so a block of keys and
// values serves the whole group and a tile's mask is as narrow as its
// 128 / group positions. Per block of 128 cached positions and tile: logits
// S = Q K^T into tensor memory (4 tcgen05.mma), a thread per row reads its 128
// logits, keeps the running maximum and sum in registers, writes the weights
// as bf16 pairs back to tensor memory, and O += P V takes them from there (8
// tcgen05.mma with V as the transposed operand, its rows as the pages hold
// them). Nothing of S or P passes through shared memory, and no row needs a
// shuffle.
//  * Outputs are rescaled only when a row's maximum has risen by more than 2^8
//    since the last time (sums and outputs carry the same reference, so the
//    quotient is exact; weights stay below 2^8).
//  * P is rounded to bf16, half a step of each weight, because the tensor
//    cores take bf16 next to V; the row's sum is kept from the unrounded ones.
//  * Softmax of one tile runs while the other's products do; q.k of the next
//    block, the next item's first among them, is issued as soon as a tile's
//    logits have been read, so items follow one another without a pause.
//  * Pages come by TMA, one copy each for keys and values, four blocks ahead;
//    a warp of its own zeroes the values of positions that no row of the item
//    sees (a weight of zero times a stale NaN would be NaN) before a block is
//    handed to the products.
__global__ void __launch_bounds__(PF_THREADS, 1)
    attn_prefill_kernel(const AttnOp a, const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                        const __grid_constant__ CUtensorMap mv, int tiles, int nx) {
    extern __shared__ __align__(16) uint8_t pf_raw[];
    uint8_t* smem = pf_raw + ((1024u - (pf_su32(pf_raw) & 1023u)) & 1023u);
    uint8_t* sq = smem;                 // [buffer][tile] of q
    uint8_t* skv = smem + 4 * PF_TILE;  // [stage][K|V]
    uint8_t* so = skv + PF_STAGES * 2 * PF_TILE;  // [tile] outputs on their way, swizzled
    uint64_t* bars = reinterpret_cast<uint64_t*>(so + 2 * PF_TILE);
    uint64_t *landed = bars, *full = bars + PF_STAGES, *empty = bars + 2 * PF_STAGES, *q_full = bars + 3 * PF_STAGES,
             *q_empty = q_full + 2, *s_full = q_full + 4, *p_ready = s_full + PF_BUFS, *o_full = p_ready + PF_BUFS;
    uint32_t* slot = reinterpret_cast<uint32_t*>(o_full + 2);
    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // known to be the same in every lane
    if (warp == 9 && lane == 0) {
        asm volatile("prefetch.tensormap [%0];\n" ::"l"(reinterpret_cast<uint64_t>(&mq)) : "memory");
        asm volatile("prefetch.tensormap [%0];\n" ::"l"(reinterpret_cast<uint64_t>(&mk)) : "memory");
        asm volatile("prefetch.tensormap [%0];\n" ::"l"(reinterpret_cast<uint64_t>(&mv)) : "memory");
    }
    const int G = a.group, per = PF_M / G, step = tiles * per;  // positions of a tile, of an item
    const int total = nx * a.kv_heads * a.seqs;

    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(pf_su32(slot)), "r"(PF_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    if (tid == 0) {
        for (int i = 0; i < PF_STAGES; i++) {
            pf_bar_init(&landed[i], 1);
            pf_bar_init(&full[i], 1);
            pf_bar_init(&empty[i], 1);
        }
        for (int t = 0; t < 2; t++) {
            pf_bar_init(&q_full[t], 1);
            pf_bar_init(&q_empty[t], 1);
            pf_bar_init(&o_full[t], 1);
        }
        for (int i = 0; i < PF_BUFS; i++) {
            pf_bar_init(&s_full[i], 1);
            pf_bar_init(&p_ready[i], 4);
        }
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    PfItems items(a, nx, total);  // the first one is on its way meanwhile
    PfItem it;
    pf_before();
    __syncthreads();
    pf_after();
    const uint32_t tmem = *slot;
    bool ok = true;
    if (warp == 8) {
        // The whole warp runs this role and one elected lane issues: the
        // descriptors then stay in uniform registers (a lone lane's products
        // went out at 71 and 57 cycles each, these at 65 and 36).
        const bool lead = pf_elect();
        const uint32_t lo_q = pf_su32(sq) >> 4, lo_kv = pf_su32(skv) >> 4;
        // the next step, a (block, tile), to compute logits for
        int nb = 0, j = 0, u = 0, stage = 0, stage_phase = 0, q = -1;
        auto next_item = [&]() {
            j = 0;
            q++;
            while (items.next(it)) {
                const PfRows rows(it, step);
                if (rows.here <= 0) continue;
                nb = rows.see(a).blocks();
                if (nb > 0) return true;
            }
            return false;
        };
        bool more = next_item();
        // The step's operands are in
        auto ready = [&]() {
            if (u) return true;
            if (j == 0 && !pf_wait_warp(&q_full[q & 1], (q >> 1) & 1)) return false;
            return pf_wait_warp(&full[stage], stage_phase);
        };
        auto logits = [&](int buf) {  // by the elected lane
            const uint32_t dq = lo_q + (uint32_t)(2 * (q & 1) + u) * (PF_TILE >> 4), dk = lo_kv + (uint32_t)stage * (2 * PF_TILE >> 4);
#pragma unroll
            for (int ks = 0; ks < 4; ks++) pf_mma_ss(tmem + buf * PF_N, pf_desc_lo(dq + 2 * ks), pf_desc_lo(dk + 2 * ks), PF_IDESC_QK, ks > 0);
            pf_commit(&s_full[buf]);
            if (u == tiles - 1 && j == nb - 1) pf_commit(&q_empty[q & 1]);
        };
        // What a step's weights' product needs, noted with its logits: stage,
        // tile, whether it adds to O, whether it is the block's last; then the
        // cursor moves on.
        auto note = [&]() {
            const bool last = u == tiles - 1;
            const int k = stage | u << 4 | (j > 0 ? 32 : 0) | (last ? 64 : 0);
            u = last ? 0 : 1;
            if (last) {
                stage = (stage + 1) % PF_STAGES;
                stage_phase ^= stage == 0;
                if (++j == nb) more = next_item();
            }
            return k;
        };
        // The steps between their two products, PF_BUFS at most, oldest first.
        // A compact loop: this warp runs its few instructions once a step,
        // between the softmax warps' long ones, and each miss in the
        // instruction cache is on the way of both.
        int note0 = -1, note1 = -1, note2 = -1;
#pragma unroll 1
        for (int buf = 0; buf < PF_BUFS; buf++) {
            if (!more) break;
            if (!(ok = ready())) break;
            pf_after();
            if (lead) logits(buf);
            __syncwarp();
            (buf == 0 ? note0 : buf == 1 ? note1 : note2) = note();
        }
        int buf = 0;
        uint32_t phase = 0;
        // Products run in the order of their issue: a step's logits follow the
        // product that read the weights in the same buffer.
#pragma unroll 1
        while (ok && note0 >= 0) {
            const bool follows = more;
            if (follows && !(ok = ready())) break;
            if (!(ok = pf_wait_warp(&p_ready[buf], phase))) break;
            pf_after();
            if (lead) {
                const uint32_t dv = lo_kv + (uint32_t)(note0 & 15) * (2 * PF_TILE >> 4) + (PF_TILE >> 4), v = (note0 >> 4) & 1;
                // a block's weights: 32 positions in 16 columns, then 16 free ones
#pragma unroll
                for (int ks = 0; ks < PF_N / 16; ks++)
                    pf_mma_ts(tmem + PF_O + v * AT_HD, tmem + buf * PF_N + (ks >> 1) * 32 + (ks & 1) * 8, pf_desc_lo(dv + ks * (2048 >> 4)),
                              PF_IDESC_PV, (note0 & 32) || ks > 0);
                pf_commit(&o_full[v]);
                if (note0 & 64) pf_commit(&empty[note0 & 15]);
                if (follows) logits(buf);
            }
            __syncwarp();
            note0 = note1;
            note1 = note2;
            note2 = follows ? note() : -1;
            if (++buf == PF_BUFS) {
                buf = 0;
                phase ^= 1;
            }
        }
    } else if (warp == 9) {
        int n = 0, q = 0;
        while (ok && items.next(it)) {
            const PfRows rows(it, step);
            if (rows.here <= 0) continue;
            const RowsSee see = rows.see(a);
            const int nb = see.blocks();
            if (nb == 0) continue;
            const int* bt = a.kv.bt + (size_t)at_seq(a.kv, it.b) * a.kv.bt_ld;
            // lanes 0-7 and 8-15 (keys, values) take a page each
            auto look_up = [&](int j) {
                const int v = j * PF_PAGES + (lane & 7);
                return v < see.np ? at_page(a.kv, bt, see.page(v), a.err) : a.kv.pages;
            };
            int page = look_up(0);
            if (q >= 2) ok = pf_wait_warp(&q_empty[q & 1], ((q >> 1) - 1) & 1);
            if (!ok) break;
            if (lane == 0) {
                pf_expect(&q_full[q & 1], (uint32_t)(tiles * per * G * 128));
                for (int u = 0; u < tiles; u++)
                    pf_copy_q(sq + (2 * (q & 1) + u) * PF_TILE, &mq, it.kh * G, it.r0 + rows.i0 + u * per, &q_full[q & 1]);
            }
            q++;
            for (int j = 0; j < nb; j++, n++) {
                const int st = n % PF_STAGES, now = page;
                if (j + 1 < nb) page = look_up(j + 1);
                if (n >= PF_STAGES && !(ok = pf_wait_warp(&empty[st], ((n / PF_STAGES) - 1) & 1))) break;
                if (lane == 0) pf_expect(&landed[st], 2 * PF_TILE);
                __syncwarp();
                if (lane < 2 * PF_PAGES)
                    pf_copy_page(skv + st * 2 * PF_TILE + (lane >> 3) * PF_TILE + (lane & 7) * (AT_PAGE * 128), lane < 8 ? &mk : &mv,
                                 it.kh, now, &landed[st]);
            }
        }
    } else if (warp == 10) {
        int n = 0;
        while (ok && items.next(it)) {
            const PfRows rows(it, step);
            if (rows.here <= 0) continue;
            const RowsSee see = rows.see(a);
            const int nb = see.blocks();
            for (int j = 0; j < nb; j++, n++) {
                const int st = n % PF_STAGES;
                if (!(ok = pf_wait_warp(&landed[st], (n / PF_STAGES) & 1))) break;
                uint8_t* tile = skv + st * 2 * PF_TILE + PF_TILE;
                for (int i = 0; i < PF_PAGES && j * PF_PAGES + i < see.np; i++) {
                    const int page = see.page(j * PF_PAGES + i);
                    if (see.all(page)) continue;
                    for (int k = lane >> 3; k < AT_PAGE; k += 4)
                        if (!see.any(page * AT_PAGE + k))
                            *reinterpret_cast<uint4*>(tile + (i * AT_PAGE + k) * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
                }
                pf_async_fence();
                __syncwarp();
                if (lane == 0) pf_arrive(&full[st]);
            }
        }
    } else if (warp < 4 * tiles) {
        const int t = warp >> 2, r = tid & 127, rp = r / G, rh = r % G;  // the tile, its row's position and head
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t to = tmem + lanes + PF_O + t * AT_HD;
        int n = 0, g0 = 0;  // blocks of this tile so far, steps of the items so far
        while (ok && items.next(it)) {
            const PfRows rows(it, step);
            if (rows.here <= 0) continue;
            const RowsSee see = rows.see(a);
            const int nb = see.blocks();
            int g = g0 + t;  // this tile's step
            g0 += nb * tiles;
            const int h = it.kh * G + rh, i = rows.i0 + t * per + rp;
            const bool has = r < per * G && t * per + rp < rows.here;
            const int pa = rows.p0 + t * per, pb = rows.p0 + min(rows.here, (t + 1) * per) - 1, p = has ? pa + rp : -1;
            const float most = 8.f / a.scale_log2;  // a rise of q.k that weights may carry (infinite at scale 0)
            float m = -INFINITY, l = 0.f;           // reference maximum (of q.k) and sum of the weights against it
            for (int j = 0; j < nb; j++, n++, g += tiles) {
                const int buf = g % PF_BUFS;
                const uint32_t ts = tmem + lanes + buf * PF_N;
                if (!(ok = pf_wait_warp(&s_full[buf], (g / PF_BUFS) & 1))) break;
                // The last item of a sequence may leave its second tile empty:
                // its steps are taken, so that every warpgroup sees every
                // phase of its barriers, but nothing is computed.
                if (pb < pa) {
                    if (j > 0 && !(ok = pf_wait_warp(&o_full[t], (n - 1) & 1))) break;
                    __syncwarp();
                    if (lane == 0) pf_arrive(&p_ready[buf]);
                    continue;
                }
                pf_after();
                const BlockSpan span(see, j);
                const bool whole = span.whole(pa, pb, a.window, a.sinks);
                uint32_t s[PF_N];
#pragma unroll
                for (int c = 0; c < PF_N; c += 32) pf_ld32(s + c, ts + c);
                pf_wait_ld(s);
                if (!whole) {
#pragma unroll
                    for (int c = 0; c < PF_N; c += 32) {
                        const uint32_t bits = span.sees(c, p, a.window, a.sinks);
                        if (__all_sync(0xffffffffu, bits == 0xffffffffu)) continue;
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
                const bool rise = top > m && (m == -INFINITY || top - m > most);
                // the last block's product has written O (waited for every
                // time: a parity names a phase only if none is left out)
                if (j > 0 && !(ok = pf_wait_warp(&o_full[t], (n - 1) & 1))) break;
                if (__any_sync(0xffffffffu, rise)) {
                    float f = 1.f;
                    if (rise) {
                        f = m == -INFINITY ? 0.f : pf_ex2((m - top) * a.scale_log2);
                        m = top;
                        l *= f;
                    }
                    if (j > 0) {
                        pf_after();
#pragma unroll 1
                        for (int c = 0; c < AT_HD; c += 16) {
                            uint32_t o[16];
                            pf_ld16(o, to + c);
                            pf_wait_ld(o);
#pragma unroll
                            for (int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                            pf_st16(to + c, o);
                        }
                    }
                }
                const float ref = m == -INFINITY ? 0.f : -m * a.scale_log2;
                const uint64_t sc2 = pf_pair(a.scale_log2, a.scale_log2), ref2 = pf_pair(ref, ref);
                uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
                for (int c = 0; c < PF_N; c += 32) {
                    uint32_t wt[16];
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        float e0, e1;
                        pf_unpair(pf_fma2(pf_pair(__uint_as_float(s[c + e]), __uint_as_float(s[c + e + 1])), sc2, ref2), e0, e1);
                        e0 = pf_ex2(e0);
                        e1 = pf_ex2(e1);
                        sum[(e >> 1) & 1] = pf_add2(sum[(e >> 1) & 1], pf_pair(e0, e1));
                        wt[e / 2] = at_bf16x2(e0, e1);
                    }
                    pf_st16(ts + c, wt);
                }
                float u0, u1;
                pf_unpair(pf_add2(sum[0], sum[1]), u0, u1);
                l += u0 + u1;
                pf_wait_st();
                pf_before();
                __syncwarp();
                if (lane == 0) pf_arrive(&p_ready[buf]);
            }
            if (ok && nb > 0) ok = pf_wait_warp(&o_full[t], (n - 1) & 1);
            pf_after();
            const float il = ok && l > 0.f ? 1.f / l : 0.f;
            // through shared memory, each warp its own 32 rows, so that eight
            // lanes store a row's 128 bytes together
            uint8_t* tile = so + t * PF_TILE + (warp & 3) * 32 * 128;
#pragma unroll
            for (int c = 0; c < AT_HD; c += 32) {
                uint32_t o[32];
                pf_ld32(o, to + c);
                pf_wait_ld(o);
#pragma unroll
                for (int e = 0; e < 32; e += 8) {
                    uint32_t y[4];
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        // nothing seen: zeros, whatever the tensor memory held
                        y[k] = l > 0.f || l != l ? at_bf16x2(__uint_as_float(o[e + 2 * k]) * il, __uint_as_float(o[e + 2 * k + 1]) * il) : 0u;
                    *reinterpret_cast<uint4*>(tile + lane * 128 + ((((c + e) / 8) ^ (lane & 7)) << 4)) = make_uint4(y[0], y[1], y[2], y[3]);
                }
            }
            __syncwarp();
            const int inv = 65536 / G + 1;  // exact below 128 for groups of at most 8
            const int first = rows.i0 + t * per, rows_of_tile = min(rows.here - t * per, per) * G;
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const int q = k * 4 + (lane >> 3), rr = (warp & 3) * 32 + q;  // a row of the tile
                const int rrp = (rr * inv) >> 16, rrh = rr - rrp * G;         // rr / G, rr % G
                const uint4 y = *reinterpret_cast<const uint4*>(tile + q * 128 + (((lane & 7) ^ (q & 7)) << 4));
                if (rr < rows_of_tile)
                    *reinterpret_cast<uint4*>(a.out + (int64_t)(it.r0 + first + rrp) * a.o_rs + (it.kh * G + rrh) * a.o_hs +
                                              (lane & 7) * 8) = y;
            }
            __syncwarp();
            if (has && a.lse)
                a.lse[(size_t)(it.r0 + i) * a.heads + h] = l == 0.f ? -INFINITY : (m * a.scale_log2 + log2f(l)) / AT_LOG2E;
            pf_before();  // the next item's products may write O once its weights are announced
        }
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
    int r0 = a.q_start[b], r1 = a.q_start[b + 1];
    at_rows(a, r0, r1);
    const int seq = at_seq(a.kv, b), n = at_len_of(a.kv, seq, a.err), first = n - (r1 - r0);
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

namespace {
constexpr int SMS = 148;

bool encode(CUtensorMap* m, const void* base, int rank, const cuuint64_t* dims, const int64_t* strides, const cuuint32_t* box) {
    using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const Encode fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
                       q == cudaDriverEntryPointSuccess
                   ? reinterpret_cast<Encode>(f)
                   : nullptr;
    }();
    if (!fn) return false;
    cuuint64_t st[4];
    // a dimension that is never stepped over may come with stride 0, which a map does not take
    for (int i = 0; i + 1 < rank; i++) st[i] = dims[i + 1] == 1 ? 16 : (cuuint64_t)strides[i] * 2;
    const cuuint32_t one[4] = {1, 1, 1, 1};
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(base), dims, st, box, one,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// K or V of one layer as [page][kv head][slot][dim], a box a page of one head
bool page_map(CUtensorMap* m, const KvPages& kv, const uint16_t* base, int kv_heads) {
    const cuuint64_t dims[4] = {AT_HD, AT_PAGE, (cuuint64_t)kv_heads, (cuuint64_t)kv.pages};
    const int64_t st[3] = {kv.ss, kv.hs, kv.ps};
    const cuuint32_t box[4] = {AT_HD, AT_PAGE, 1, 1};
    return encode(m, base, 4, dims, st, box);
}
// q as [row][head][dim], a box the heads of a group at `per` rows
bool q_map(CUtensorMap* m, const AttnOp& a, int per) {
    const cuuint64_t dims[3] = {AT_HD, (cuuint64_t)a.heads, (cuuint64_t)a.rows};
    const int64_t st[2] = {a.q_hs, a.q_rs};
    const cuuint32_t box[3] = {AT_HD, (cuuint32_t)a.group, (cuuint32_t)per};
    return encode(m, a.q, 3, dims, st, box);
}
}  // namespace

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
    const int per = PF_M / a.group;
    CUtensorMap mq, mk, mv;
    if (!q_map(&mq, a, per) || !page_map(&mk, a.kv, a.kv.k, a.kv_heads) || !page_map(&mv, a.kv, a.kv.v, a.kv_heads))
        return cudaErrorInvalidValue;
    // items of one tile while every one of them finds an SM: the latency of a
    // block is then one tile's
    const long long heads = (long long)a.kv_heads * a.seqs, one = (long long)((a.max_rows + per - 1) / per) * heads;
    const int tiles = one <= SMS ? 1 : 2;
    const int nx = (a.max_rows + tiles * per - 1) / (tiles * per);
    if (nx * heads > 0x7fffffff) return cudaErrorInvalidValue;
    const int grid = (int)std::min<long long>(SMS, nx * heads);
    attn_prefill_kernel<<<grid, PF_THREADS, PF_SMEM, s>>>(a, mq, mk, mv, tiles, nx);
    return cudaGetLastError();
}

cudaError_t launch_attn_weights(const AttnOp& a, cudaStream_t s) {
    attn_weights_kernel<<<dim3((a.kv.max_len + 127) / 128, a.kv_heads, a.seqs), 128, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace ming
