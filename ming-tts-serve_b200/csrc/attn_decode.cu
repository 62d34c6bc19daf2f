// attn_decode.cu — attention of one new token per sequence over a paged cache.
#include <cuda_runtime.h>

#include "attn.cuh"

namespace ming {

// One warp per (row, kv head): each lane holds two dims, a position's dot is a
// warp sum. The simple form that every later one is checked against.
__global__ void __launch_bounds__(32) attn_decode_kernel(const AttnOp a) {
    const int b = blockIdx.x, kh = blockIdx.y, lane = threadIdx.x;
    const int seq = at_seq(a.kv, b), n = at_len(a.kv, seq, a.err), p = n - 1;
    const int* bt = a.kv.bt + (size_t)seq * a.kv.bt_ld;
    int s1, w0;
    at_sees(p, a.window, a.sinks, s1, w0);
    auto row = [&](const uint16_t* base, int j) {
        return base + (int64_t)at_page(a.kv, bt, j / AT_PAGE, a.err) * a.kv.ps + kh * a.kv.hs + (j % AT_PAGE) * a.kv.ss;
    };
    float q[AT_MAXG][2], m[AT_MAXG], l[AT_MAXG], o[AT_MAXG][2];
    for (int g = 0; g < AT_MAXG; g++) {
        const uint16_t* qr = a.q + b * a.q_rs + (kh * a.group + (g < a.group ? g : 0)) * a.q_hs;
        q[g][0] = bf2f(qr[2 * lane]) * a.scale_log2;
        q[g][1] = bf2f(qr[2 * lane + 1]) * a.scale_log2;
        m[g] = -INFINITY;
        l[g] = o[g][0] = o[g][1] = 0.f;
    }
    for (int pass = 0; pass < (a.acc ? 2 : 1); pass++)
        for (int j = 0; j < n; j++) {
            if (j == s1) j = w0;
            if (j >= n) break;
            const float2 k = unpack_bf16x2(reinterpret_cast<const uint32_t*>(row(a.kv.k, j))[lane]);
            const float2 v = unpack_bf16x2(reinterpret_cast<const uint32_t*>(row(a.kv.v, j))[lane]);
            float w = 0.f;
            for (int g = 0; g < a.group; g++) {
                const float s = warp_sum(q[g][0] * k.x + q[g][1] * k.y);
                if (pass == 0) {
                    const float mn = fmaxf(m[g], s), c = exp2f(m[g] - mn), e = exp2f(s - mn);
                    m[g] = mn;
                    l[g] = l[g] * c + e;
                    o[g][0] = o[g][0] * c + e * v.x;
                    o[g][1] = o[g][1] * c + e * v.y;
                } else {
                    w += exp2f(s - m[g]) / l[g];
                }
            }
            if (pass == 1 && lane == 0) {
                float* t = a.acc + seq * a.a_ss + kh * a.a_hs + j;
                *t = (j == p ? 0.f : *t) + w;
            }
        }
    for (int g = 0; g < a.group; g++) {
        const float il = l[g] > 0.f ? 1.f / l[g] : 0.f;
        reinterpret_cast<uint32_t*>(a.out + b * a.o_rs + (kh * a.group + g) * a.o_hs)[lane] =
            pack_bf16x2(o[g][0] * il, o[g][1] * il);
    }
}

cudaError_t launch_attn_decode(const AttnOp& a, cudaStream_t s) {
    attn_decode_kernel<<<dim3(a.seqs, a.kv_heads), 32, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace ming
