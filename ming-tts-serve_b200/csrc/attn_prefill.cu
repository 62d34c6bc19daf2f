// attn_prefill.cu — attention of a prompt's rows over a paged cache, and the
// weights that those rows gave to each cached position.
#include <cuda_runtime.h>

#include "attn.cuh"

namespace ming {

// One warp per (row of a sequence, head): each lane holds two dims. The simple
// form that every later one is checked against.
__global__ void __launch_bounds__(32) attn_prefill_kernel(const AttnOp a) {
    const int b = blockIdx.z, h = blockIdx.y, lane = threadIdx.x, kh = h / a.group;
    int r0, r1;
    at_rows(a, b, r0, r1);
    const int r = r0 + blockIdx.x;
    if (r >= r1) return;
    const int seq = at_seq(a.kv, b), n = at_len(a.kv, seq, a.err), p = n - (r1 - r);
    const int* bt = a.kv.bt + (size_t)seq * a.kv.bt_ld;
    int s1, w0;
    at_sees(p, a.window, a.sinks, s1, w0);
    const uint16_t* qr = a.q + r * a.q_rs + h * a.q_hs;
    const float q0 = bf2f(qr[2 * lane]) * a.scale_log2, q1 = bf2f(qr[2 * lane + 1]) * a.scale_log2;
    float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
    for (int j = 0; j <= p; j++) {
        if (j == s1) j = w0;
        if (j > p) break;
        const int64_t at = (int64_t)at_page(a.kv, bt, j / AT_PAGE, a.err) * a.kv.ps + kh * a.kv.hs + (j % AT_PAGE) * a.kv.ss;
        const float2 k = unpack_bf16x2(reinterpret_cast<const uint32_t*>(a.kv.k + at)[lane]);
        const float2 v = unpack_bf16x2(reinterpret_cast<const uint32_t*>(a.kv.v + at)[lane]);
        const float s = warp_sum(q0 * k.x + q1 * k.y);
        const float mn = fmaxf(m, s), c = exp2f(m - mn), e = exp2f(s - mn);
        m = mn;
        l = l * c + e;
        o0 = o0 * c + e * v.x;
        o1 = o1 * c + e * v.y;
    }
    const float il = l > 0.f ? 1.f / l : 0.f;
    reinterpret_cast<uint32_t*>(a.out + r * a.o_rs + h * a.o_hs)[lane] = pack_bf16x2(o0 * il, o1 * il);
    if (a.lse && lane == 0) a.lse[(size_t)r * a.heads + h] = l > 0.f ? (m + log2f(l)) / AT_LOG2E : -INFINITY;
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
    attn_prefill_kernel<<<dim3(a.max_rows, a.heads, a.seqs), 32, 0, s>>>(a);
    return cudaGetLastError();
}

cudaError_t launch_attn_weights(const AttnOp& a, cudaStream_t s) {
    attn_weights_kernel<<<dim3((a.kv.max_len + 127) / 128, a.kv_heads, a.seqs), 128, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace ming
