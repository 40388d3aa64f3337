// Attention over the 4-bit cache (csrc/kv4.cuh).
#include <cuda_fp16.h>

#include "common.cuh"
#include "kv4.cuh"

namespace alice {

// A warp a row: (token, query head). Lane l holds dims l, l + 32, ...
__global__ void __launch_bounds__(32) kv4_attn_kernel(const __grid_constant__ Kv4AttnArgs a) {
    pdl_launch_dependents();
    pdl_wait();
    const Kv4Plan& pl = a.plan;
    const uint32_t lane = threadIdx.x, head = blockIdx.y, dim = a.shape.dim, nb = dim / KV4_BLOCK;
    const Kv4Head hd = *pl.head;
    if (!kv4_fits(hd, a.most_tokens, a.rope, a.shape, gridDim.z, a.status) || blockIdx.x >= hd.jobs) return;
    const uint32_t seq = pl.job_seq[blockIdx.x], row = pl.job_row[blockIdx.x] + blockIdx.z;
    if (row >= pl.seq_count[seq] * a.group) return;
    const uint32_t tok = row / a.group, qh = head * a.group + row % a.group, at = pl.seq_first[seq] + tok, pos = pl.seq_past[seq] + tok;
    const float* q = a.q + at * a.q_ld + (size_t)qh * dim;
    const float* turn = a.rope.table + (size_t)(a.rope.by_token ? at : pos) * a.rope.dims;
    float x[8], o[8], mx = -INFINITY, sum = 0;
    for (uint32_t b = 0; b < nb; b++) {
        const uint32_t d = b * 32 + lane, half = a.rope.dims / 2;
        x[b] = q[d]; o[b] = 0;
        if (d < a.rope.dims) {
            const bool upper = a.rope.neox ? d >= half : d & 1;
            const uint32_t j = a.rope.neox ? d % half : d / 2, other = a.rope.neox ? (upper ? d - half : d + half) : d ^ 1;
            x[b] = upper ? q[other] * turn[2 * j] + x[b] * turn[2 * j + 1] : x[b] * turn[2 * j + 1] - q[other] * turn[2 * j];
        }
    }
    for (uint32_t j = 0; j <= pos; j++) {
        const uint32_t page = pl.table[(size_t)seq * pl.table_ld + j / a.shape.page_tokens], in_page = j % a.shape.page_tokens, p = in_page % KV4_TILE, r = kv4_row(p);
        const uint8_t* tile = a.pool + (((size_t)page * a.shape.kv_heads + head) * a.shape.tiles() + in_page / KV4_TILE) * kv4_tile_bytes(dim);
        float s = 0, v[8];
        for (uint32_t b = 0; b < nb; b++) {
            const uint32_t kc = *reinterpret_cast<const uint32_t*>(tile + r * (dim / 2) + kv4_k_word(nb, b, lane / 8) * 4) >> (4 * (lane % 8)) & 15;
            const uint32_t vc = *reinterpret_cast<const unsigned short*>(tile + kv4_v_codes(dim) + p * (dim / 2) + (lane / 4 * nb + b) * 2) >> (4 * (lane % 4)) & 15;
            const float2 ks = __half22float2(*reinterpret_cast<const __half2*>(tile + kv4_k_scales(dim) + (r * nb + b) * 4));
            const float2 vs = __half22float2(*reinterpret_cast<const __half2*>(tile + kv4_v_scales(dim) + (r * nb + b) * 4));
            s += x[b] * (ks.x * kc + ks.y);
            v[b] = vs.x * vc + vs.y;
        }
        s = warp_sum(s) * a.scale;
        const float m = fmaxf(mx, s), c = m == -INFINITY ? 1.f : expf(mx - m), w = m == -INFINITY ? 0.f : expf(s - m);
        sum = sum * c + w; mx = m;
        for (uint32_t b = 0; b < nb; b++) o[b] = o[b] * c + w * v[b];
    }
    for (uint32_t b = 0; b < nb; b++) a.out[at * a.out_ld + (size_t)qh * dim + b * 32 + lane] = o[b] / sum;
}

size_t kv4_part_floats(uint32_t, int) { return 1; }

cudaError_t launch_kv4_attention(const Kv4AttnArgs& a, uint32_t rows, uint32_t jobs, int, cudaStream_t st, bool pdl) {
    if (!jobs) return cudaSuccess;
    cudaLaunchConfig_t lc = {}; cudaLaunchAttribute at[1];
    lc.gridDim = dim3(jobs, a.shape.kv_heads, rows); lc.blockDim = dim3(32); lc.stream = st;
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = at; lc.numAttrs = pdl ? 1 : 0;
    return cudaLaunchKernelEx(&lc, kv4_attn_kernel, a);
}

}  // namespace alice
