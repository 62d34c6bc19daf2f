// attn_weights.cu — the attention weights that a prompt's rows gave to each
// cached position, on the 5th-generation tensor cores.
#include <cuda_runtime.h>

#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>

#include "attn_tc.cuh"

namespace ming {

namespace {
namespace cg = cooperative_groups;

constexpr int WT_STAGES = 2;
constexpr int WT_THREADS = 192;  // four warps of weights, one of products, one of copies
constexpr int WT_PER_SM = 4;
constexpr int WT_MAX_SPLIT = 16;  // CTAs of a cluster
constexpr int WT_OWNERS = 4;      // ranks that add up the sums of a quarter of the positions each
constexpr int WT_LSE = AT_M * 4;
constexpr int WT_SMEM = 1024 + AT_TILE + WT_STAGES * AT_TILE + WT_STAGES * WT_LSE + 128 + WT_MAX_SPLIT * AT_N / WT_OWNERS * 4;
}  // namespace

// acc[j] (+)= sum over rows i and the group's heads of exp(s_ij - lse_i).
// The transposed product S^T = K Q^T puts a cached position on each of the 128
// rows of the tile and 128 (position, head) rows of q on its columns: a thread
// owns one cached position and adds up its columns, so that no sum crosses
// threads. lse (times -log2 e) comes along the columns from shared memory,
// minus infinity where a column is no row.
// A cluster takes a tile of 128 cached positions of one (sequence, kv head);
// its CTAs split the tiles of q that see it, and their sums go through distributed
// shared memory to the first ranks, which add them up rank by rank while the
// others leave: no atomics, one order of sums.
// Bound by the exponentials, 16 a cycle and SM, one per visible pair: four
// CTAs share an SM (128 tensor memory columns and 55 KB each) and fill each
// other's waits, so each keeps one buffer of logits and two tiles of q.
// Measured: 8 prompts of up to 2048 rows (14 query, 2 kv heads) 56.6 us, the
// exponential unit 46% busy: at its rate inside the loop, but a CTA's start
// (its first logits 3 us after launch) and end take a third of its time. One
// prompt of 333 rows: 7.4 us. Slower: two tiles of positions a cluster, from
// both ends (78 us), three CTAs an SM with three tiles of q each (63).
__global__ void __launch_bounds__(WT_THREADS, WT_PER_SM)
    attn_weights_kernel(const AttnOp a, const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk, int split) {
    extern __shared__ __align__(16) uint8_t wt_raw[];
    uint8_t* smem = wt_raw + ((1024u - (at_su32(wt_raw) & 1023u)) & 1023u);
    uint8_t *sk = smem, *sq = smem + AT_TILE;
    float* nlse = reinterpret_cast<float*>(sq + WT_STAGES * AT_TILE);  // [stage][column]
    uint64_t *k_full = reinterpret_cast<uint64_t*>(nlse + WT_STAGES * AT_M), *q_full = k_full + 1,
             *q_empty = q_full + WT_STAGES, *s_full = q_empty + WT_STAGES, *s_read = s_full + 1;
    uint32_t* slot = reinterpret_cast<uint32_t*>(s_read + 1);
    float* part = reinterpret_cast<float*>(slot + 4);  // an owner's: [rank][AT_N / owners], all ranks' sums of its positions
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    // the first tiles of every sequence, which the most rows see, start first
    const int rank = blockIdx.x % split, kh = blockIdx.x / split % a.kv_heads, b = blockIdx.x / split / a.kv_heads, tile = blockIdx.y;
    const int G = a.group, per = AT_M / G;
    const int seq = at_seq(a.kv, b);
    int r0 = a.q_start[b], r1 = a.q_start[b + 1];
    const int held = a.kv.lens[seq] + a.kv.len_add;
    if (warp == 5 && lane == 0) {
        asm volatile("prefetch.tensormap [%0];\n" ::"l"(reinterpret_cast<uint64_t>(&mq)) : "memory");
        asm volatile("prefetch.tensormap [%0];\n" ::"l"(reinterpret_cast<uint64_t>(&mk)) : "memory");
    }
    at_rows(a, r0, r1);
    const int len = at_len(a.kv, held, a.err), rows = r1 - r0, first = len - rows;
    // the rows of the sequence that see any position of the tile, and this CTA's share of them
    const int j0 = tile * AT_N, lo = max(0, j0 - first), last = min(j0 + AT_N, len) - 1;
    const int hi = a.window && j0 >= a.sinks ? (int)min((long long)rows, (long long)last + a.window - first) : rows;
    if (j0 >= len || lo >= hi) return;  // the whole cluster
    // This CTA runs: the others may write to its memory once all have said so.
    // (Said before tensor memory is asked for, so that no one holds any while
    // it waits for a CTA that cannot get some.)
    if (split > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
    const int nt = (hi - lo + per - 1) / per, t0 = (int)((long long)nt * rank / split), steps = (int)((long long)nt * (rank + 1) / split) - t0;

    if (warp == 4) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(at_su32(slot)), "r"(AT_N) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    // The copying warp sets the barriers up and starts its first copies without
    // waiting for the others.
    auto copy_q = [&](int s) {
        const int st = s % WT_STAGES;
        at_expect(&q_full[st], (uint32_t)(per * G * 128));
        at_copy_q(sq + st * AT_TILE, &mq, kh * G, r0 + lo + (t0 + s) * per, &q_full[st]);
    };
    if (warp == 5) {
        int page = a.kv.pages;
        if (lane < AT_BLOCK_PAGES && j0 / AT_PAGE + lane < (len + AT_PAGE - 1) / AT_PAGE)
            page = at_page(a.kv, a.kv.bt + (size_t)seq * a.kv.bt_ld, j0 / AT_PAGE + lane, a.err);
        if (lane == 0) {
            at_bar_init(k_full, 1);
            for (int i = 0; i < WT_STAGES; i++) {
                at_bar_init(&q_full[i], 2);
                at_bar_init(&q_empty[i], 5);
            }
            at_bar_init(s_full, 1);
            at_bar_init(s_read, 4);
            asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
            at_async_fence();
            for (int s = 0; s < min(steps, WT_STAGES); s++) copy_q(s);
            if (steps > 0) at_expect(k_full, AT_TILE);
        }
        __syncwarp();
        if (steps > 0 && lane < AT_BLOCK_PAGES) at_copy_page(sk + lane * (AT_PAGE * 128), &mk, kh, page, k_full);
    } else {
        // columns that the copies never reach
        const int tail = (AT_M - per * G) * 8;
        for (int e = tid; e < WT_STAGES * tail; e += WT_THREADS - 32)
            *reinterpret_cast<uint4*>(sq + e / tail * AT_TILE + (per * G + e % tail / 8) * 128 + (e % 8) * 16) = make_uint4(0, 0, 0, 0);
    }
    at_async_fence();
    at_before();
    __syncthreads();
    at_after();
    const uint32_t tmem = *slot;
    bool ok = true;
    float total = 0.f;
    if (warp == 4) {
        const bool lead = at_elect();
        const uint32_t dk = at_su32(sk) >> 4, dq = at_su32(sq) >> 4;
        if (steps > 0) ok = at_wait_warp(k_full, 0);
#pragma unroll 1
        for (int s = 0; ok && s < steps; s++) {
            const int st = s % WT_STAGES;
            if (!(ok = at_wait_warp(&q_full[st], (s / WT_STAGES) & 1))) break;
            if (s > 0 && !(ok = at_wait_warp(s_read, (s - 1) & 1))) break;
            at_after();
            if (lead) {
#pragma unroll
                for (int ks = 0; ks < 4; ks++)
                    at_mma_ss(tmem, at_desc_lo(dk + 2 * ks), at_desc_lo(dq + st * (AT_TILE >> 4) + 2 * ks), AT_IDESC_QK, ks > 0);
                at_commit(s_full);
                at_commit(&q_empty[st]);
            }
            __syncwarp();
        }
    } else if (warp == 5) {
        // a column's row and head, the same in every tile
        int off[AT_M / 32];
#pragma unroll
        for (int k = 0; k < AT_M / 32; k++) off[k] = (k * 32 + lane) / G * a.heads + kh * G + (k * 32 + lane) % G;
#pragma unroll 1
        for (int s = 0; s < steps; s++) {
            const int st = s % WT_STAGES, i0 = lo + (t0 + s) * per, m = min(per, rows - i0) * G;  // columns that are rows
            if (s >= WT_STAGES) {
                if (!(ok = at_wait_warp(&q_empty[st], ((s / WT_STAGES) - 1) & 1))) break;
                if (lane == 0) copy_q(s);
            }
            const float* from = a.lse + (size_t)(r0 + i0) * a.heads;
#pragma unroll
            for (int k = 0; k < AT_M / 32; k++)
                nlse[st * AT_M + k * 32 + lane] = k * 32 + lane < m ? -AT_LOG2E * from[off[k]] : -INFINITY;
            __syncwarp();
            if (lane == 0) at_arrive(&q_full[st]);
        }
    } else {
        const uint32_t ts = tmem + ((uint32_t)(warp * 32) << 16);
        const uint64_t sc2 = at_pair(a.scale_log2, a.scale_log2);
        const int j = j0 + tid;
#pragma unroll 1
                    for (int s = 0; s < steps; s++) {
                        const int st = s % WT_STAGES, i0 = lo + (t0 + s) * per;
                        // the tile's rows that see position j, as columns; everyone's, if no one leaves any out
                        const int c_lo = max(0, j - first - i0) * G;
                        const int seen = a.window && j >= a.sinks ? (int)min((long long)per, (long long)j + a.window - first - i0) : per;
                        const int c_hi = max(0, min(min(per, rows - i0), seen)) * G;
                        const bool whole = __all_sync(0xffffffffu, c_lo == 0 && c_hi == per * G);
                        if (!(ok = at_wait_warp(s_full, s & 1))) break;
                        at_after();
                        uint64_t sum[2] = {0ull, 0ull};
                        const float* nl = nlse + st * AT_M;
#pragma unroll 1
                        for (int c = 0; c < AT_M; c += 32) {
                            uint32_t v[32];
                            at_ld32(v, ts + c);
                            at_wait_ld(v);
                            if (c == AT_M - 32) {
                                at_before();
                                __syncwarp();
                                if (lane == 0) at_arrive(s_read);
                            }
                            if (!whole) {
                                const uint32_t bits = at_bits(c_lo - c, c_hi - c);
#pragma unroll
                                for (int e = 0; e < 32; e++)
                                    if (!((bits >> e) & 1u)) v[e] = 0xff800000u;  // -infinity
                            }
#pragma unroll
                            for (int e = 0; e < 32; e += 4) {
                                const ulonglong2 z = *reinterpret_cast<const ulonglong2*>(nl + c + e);
                                float x0, x1, x2, x3;
                                at_unpair(at_fma2(at_pair(__uint_as_float(v[e]), __uint_as_float(v[e + 1])), sc2, z.x), x0, x1);
                                at_unpair(at_fma2(at_pair(__uint_as_float(v[e + 2]), __uint_as_float(v[e + 3])), sc2, z.y), x2, x3);
                                sum[0] = at_add2(sum[0], at_pair(at_ex2(x0), at_ex2(x1)));
                                sum[1] = at_add2(sum[1], at_pair(at_ex2(x2), at_ex2(x3)));
                            }
                        }
                        float u0, u1;
                        at_unpair(at_add2(sum[0], sum[1]), u0, u1);
                        total += u0 + u1;
                        __syncwarp();
                        if (lane == 0) at_arrive(&q_empty[st]);
                    }
    }
    if (!ok) at_flag(a.err, AT_ERR_WAIT);
    cg::cluster_group cluster = cg::this_cluster();
    if (split > 1) asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
    const int owners = min(split, WT_OWNERS), share = AT_N / owners;
    if (warp < 4) (split > 1 ? cluster.map_shared_rank(part, tid / share) : part)[rank * share + tid % share] = total;
    // tensor memory back before the cluster's barrier
    at_before();
    __syncthreads();
    if (warp == 4) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(AT_N) : "memory");
    if (split > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
    if (rank >= owners) return;
    if (split > 1) asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
    for (int e = tid; e < share; e += WT_THREADS) {
        const int t = rank * share + e;
        float w = 0.f;
        for (int q = 0; q < split; q++) w += part[q * share + e];
        const int j = j0 + t;
        if (j < len) {
            float* d = a.acc + seq * a.a_ss + kh * a.a_hs + j;
            *d = (j >= first ? 0.f : *d) + w;
        }
    }
}

cudaError_t launch_attn_weights(const AttnOp& a, cudaStream_t s) {
    static std::atomic<bool> ready[64] = {};  // per device: the kernel's attributes are set
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !ready[dev].load(std::memory_order_acquire)) {
        if ((e = cudaFuncSetAttribute(attn_weights_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, WT_SMEM)) != cudaSuccess) return e;
        if ((e = cudaFuncSetAttribute(attn_weights_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1)) != cudaSuccess) return e;
        if (dev < 64) ready[dev].store(true, std::memory_order_release);
    }
    const int per = AT_M / a.group;
    CUtensorMap mq, mk;
    if (!at_q_map(&mq, a, per) || !at_page_map(&mk, a.kv, a.kv.k, a.kv_heads)) return cudaErrorInvalidValue;
    // splits: two rounds of CTAs for every SM's four places, if each still has a few tiles of q
    const int tiles = (a.kv.max_len + AT_N - 1) / AT_N, nq = (a.max_rows + per - 1) / per;
    if (tiles > 65535 || 16ll * a.kv_heads * a.seqs > 0x7fffffff) return cudaErrorInvalidValue;
    int split = 1;
    while (split < WT_MAX_SPLIT && (long long)tiles * a.kv_heads * a.seqs * split < 2ll * AT_SMS * WT_PER_SM && nq > 2 * split) split *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(split * a.kv_heads * a.seqs, tiles);
    cfg.blockDim = dim3(WT_THREADS);
    cfg.dynamicSmemBytes = WT_SMEM;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = split;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, attn_weights_kernel, a, mq, mk, split);
}

}  // namespace ming
