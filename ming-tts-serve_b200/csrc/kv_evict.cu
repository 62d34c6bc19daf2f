// kv_evict.cu — eviction from a paged K/V cache by accumulated attention weight.
#include <cuda_runtime.h>

#include "attn.cuh"

namespace ming {

namespace {
constexpr int EV_THREADS = 256;

// Order-preserving key of a total: larger total, larger key. -0 counts as +0
// and NaN as -infinity.
MING_DEV uint32_t ev_key(float x) {
    if (isnan(x)) x = -INFINITY;
    const uint32_t u = __float_as_uint(x + 0.f);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
}  // namespace

// One CTA per (sequence, layer, kv head). Which positions stay: the first
// `sinks`, the last `recent`, and of those between the keep - sinks - recent
// of the largest total. The smallest total that stays is found digit by digit
// (four passes of 8 bits over the keys, a histogram each); positions that tie
// with it stay from the lowest on. Then the positions are walked in blocks of
// EV_THREADS: the block's kept rows are read, and after a barrier written to
// their places. A row's place is never behind it, so a block never overwrites
// what a later one reads, and the move may be in place.
__global__ void __launch_bounds__(EV_THREADS) kv_evict_kernel(const EvictOp a) {
    __shared__ int hist[256];
    __shared__ uint32_t s_prefix;
    __shared__ int s_need, warp_kept[8], warp_ties[8], kept_pos[EV_THREADS];
    const int b = blockIdx.z, layer = blockIdx.y, kh = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int seq = at_seq(a.from, b), n = at_len_of(a.from, seq, a.err), keep = min(a.keep, n);
    const int lo = min(a.sinks, n), hi = max(lo, n - a.recent), need = n > a.keep ? a.keep - lo - (n - hi) : hi - lo;
    const float* acc = a.acc ? a.acc + seq * a.a_ss + layer * a.a_ls + kh * a.a_hs : nullptr;
    float* acc_to = a.acc_to ? a.acc_to + seq * a.t_ss + layer * a.t_ls + kh * a.t_hs : nullptr;
    uint32_t cut = 0;   // positions between with a key above it stay
    int ties = hi - lo; // and so many of those at it
    if (need < hi - lo) {
        if (need > 0) {
            uint32_t prefix = 0;
            int left = need;
            for (int shift = 24; shift >= 0; shift -= 8) {
                hist[tid] = 0;
                __syncthreads();
                for (int j = lo + tid; j < hi; j += EV_THREADS) {
                    const uint32_t k = ev_key(acc[j]);
                    if (shift == 24 || (k >> (shift + 8)) == prefix) atomicAdd(&hist[(k >> shift) & 255], 1);
                }
                __syncthreads();
                if (tid == 0) {
                    int d = 255, above = 0;
                    while (d > 0 && above + hist[d] < left) above += hist[d--];
                    s_prefix = (prefix << 8) | (uint32_t)d;
                    s_need = left - above;
                }
                __syncthreads();
                prefix = s_prefix;
                left = s_need;
            }
            cut = prefix;
            ties = left;
        } else {
            cut = 0xffffffffu;
            ties = 0;
        }
    }
    const bool all = need >= hi - lo, none = need <= 0;
    const int* bt = a.from.bt + (size_t)seq * a.from.bt_ld;
    const int* bt_to = a.to.bt + (size_t)seq * a.to.bt_ld;
    int slot0 = 0, ties0 = 0;  // kept, and ties seen, before this block
    for (int j0 = 0; j0 < n; j0 += EV_THREADS) {
        const int j = j0 + tid;
        const bool mid = j >= lo && j < hi;
        const uint32_t k = mid && !all && !none ? ev_key(acc[j]) : 0;
        const bool tie = mid && !all && !none && k == cut;
        const unsigned bt_tie = __ballot_sync(0xffffffffu, tie);
        if (lane == 0) warp_ties[warp] = __popc(bt_tie);
        __syncthreads();
        int t = ties0 + __popc(bt_tie & ((1u << lane) - 1));
        for (int w = 0; w < warp; w++) t += warp_ties[w];
        const bool stays = j < n && (!mid || all || (!none && (k > cut || (tie && t < ties))));
        const unsigned bs = __ballot_sync(0xffffffffu, stays);
        if (lane == 0) warp_kept[warp] = __popc(bs);
        __syncthreads();
        int slot = __popc(bs & ((1u << lane) - 1)), total = 0;
        for (int w = 0; w < 8; w++) {
            if (w < warp) slot += warp_kept[w];
            total += warp_kept[w];
            ties0 += warp_ties[w];
        }
        if (stays) kept_pos[slot] = j;
        const float av = stays && acc ? acc[j] : 0.f;
        __syncthreads();
        // the block's rows: K then V, eight 16-byte parts each
        for (int which = 0; which < 2; which++) {
            uint4 v[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int e = tid + i * EV_THREADS, s = e >> 3;
                if (s < total) {
                    const int p = kept_pos[s];
                    const uint16_t* src = (which ? a.from.v : a.from.k) + layer * a.from_ls +
                                          (int64_t)at_page(a.from, bt, p / AT_PAGE, a.err) * a.from.ps + kh * a.from.hs +
                                          (p % AT_PAGE) * a.from.ss;
                    v[i] = reinterpret_cast<const uint4*>(src)[e & 7];
                }
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int e = tid + i * EV_THREADS, s = e >> 3;
                if (s < total) {
                    const int p = slot0 + s, page = bt_to[p / AT_PAGE];
                    if ((unsigned)page < (unsigned)a.to.pages)
                        reinterpret_cast<uint4*>((which ? a.to.v : a.to.k) + layer * a.to_ls + (int64_t)page * a.to.ps +
                                                 kh * a.to.hs + (p % AT_PAGE) * a.to.ss)[e & 7] = v[i];
                    else
                        at_flag(a.err, AT_ERR_PAGE);
                }
            }
        }
        if (stays) {
            if (acc_to) acc_to[slot0 + slot] = av;
            if (a.index) a.index[(((size_t)b * a.layers + layer) * a.kv_heads + kh) * a.keep + slot0 + slot] = j;
        }
        slot0 += total;
        __syncthreads();
    }
    if (a.index)
        for (int s = keep + tid; s < a.keep; s += EV_THREADS)
            a.index[(((size_t)b * a.layers + layer) * a.kv_heads + kh) * a.keep + s] = -1;
}

cudaError_t launch_kv_evict(const EvictOp& a, cudaStream_t s) {
    kv_evict_kernel<<<dim3(a.kv_heads, a.layers, a.seqs), EV_THREADS, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace ming
