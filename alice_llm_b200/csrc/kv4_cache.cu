// Rows of keys and values into and out of the 4-bit cache (csrc/kv4.cuh).
#include <cuda_fp16.h>

#include "common.cuh"
#include "kv4.cuh"

namespace alice {

namespace {

// Eight lanes hold one block of 32 values of one row, four values each.
struct RowPlace {
    uint32_t tok, head, block, sub;
    bool value, in;
};
__device__ __forceinline__ RowPlace row_place(uint32_t i, uint32_t n, const Kv4Shape& s) {
    RowPlace p;
    const uint32_t nb = s.dim / KV4_BLOCK, unit = i >> 3;
    p.sub = i & 7;
    p.block = unit % nb;
    const uint32_t r = unit / nb;
    p.value = r & 1;
    p.head = (r >> 1) % s.kv_heads;
    p.tok = (r >> 1) / s.kv_heads;
    p.in = p.tok < n;
    if (!p.in) p.tok = 0;
    return p;
}
// The 4 codes (16 bits) and the scales of a lane's values within the tile of the position in `slot`.
struct CodePlace { size_t codes, scales; };
__device__ __forceinline__ CodePlace code_place(const RowPlace& p, uint32_t slot, const Kv4Shape& s) {
    const uint32_t nb = s.dim / KV4_BLOCK, page = slot / s.page_tokens, in_page = slot % s.page_tokens, pos = in_page % KV4_TILE, row = kv4_row(pos);
    const size_t tile = (((size_t)page * s.kv_heads + p.head) * s.tiles() + in_page / KV4_TILE) * kv4_tile_bytes(s.dim);
    CodePlace c;
    c.codes = tile + (p.value ? kv4_v_codes(s.dim) + pos * (s.dim / 2) + (p.sub * nb + p.block) * 2
                              : row * (s.dim / 2) + kv4_k_word(nb, p.block, p.sub >> 1) * 4 + (p.sub & 1) * 2);
    c.scales = tile + (p.value ? kv4_v_scales(s.dim) : kv4_k_scales(s.dim)) + row * (4 * nb) + p.block * 2;     // d; m is 2 nb further
    return c;
}

__device__ __forceinline__ double max8(double v) {
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

}  // namespace

// Keys are rotated and everything is put into codes in f64: the products of f32 numbers are exact there, and a value that lies on the
// border of two codes goes where the formula says.
__global__ void __launch_bounds__(256) kv4_append_kernel(const __grid_constant__ Kv4RowsArgs a) {
    pdl_launch_dependents();
    pdl_wait();
    const Kv4Head head = *a.plan.head;
    if (!kv4_fits(head, a.most_tokens, a.rope, a.shape, 0, a.status)) return;
    const uint32_t n = head.tokens, nb = a.shape.dim / KV4_BLOCK;
    const uint32_t lanes = n * a.shape.kv_heads * 2 * nb * 8;
    for (uint32_t i0 = blockIdx.x * 256; i0 < lanes; i0 += gridDim.x * 256) {
        const RowPlace p = row_place(i0 + threadIdx.x, n, a.shape);
        const uint32_t dim0 = p.block * KV4_BLOCK + p.sub * 4;
        const float* row = (p.value ? a.v + p.tok * a.v_ld : a.k + p.tok * a.k_ld) + (size_t)p.head * a.shape.dim;
        const float4 f = __ldg(reinterpret_cast<const float4*>(row + dim0));
        double x[4] = {f.x, f.y, f.z, f.w};
        if (!p.value && dim0 < a.rope.dims) {
            const float* turn = a.rope.table + (size_t)(a.rope.by_token ? p.tok : a.plan.tok_pos[p.tok]) * a.rope.dims;
            if (a.rope.neox) {
                const uint32_t half = a.rope.dims / 2;
                const bool upper = dim0 >= half;
                const uint32_t j = upper ? dim0 - half : dim0;
                const float4 o = __ldg(reinterpret_cast<const float4*>(row + (upper ? j : dim0 + half)));
                const float other[4] = {o.x, o.y, o.z, o.w};
                const float4 w0 = __ldg(reinterpret_cast<const float4*>(turn + 2 * j)), w1 = __ldg(reinterpret_cast<const float4*>(turn + 2 * j + 4));
                const float sn[4] = {w0.x, w0.z, w1.x, w1.z}, cs[4] = {w0.y, w0.w, w1.y, w1.w};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const double t = __dmul_rn((double)other[e], (double)sn[e]);     // exact; one rounding in the sum
                    x[e] = __dadd_rn(__dmul_rn(x[e], (double)cs[e]), upper ? t : -t);
                }
            } else {
                const float4 w = __ldg(reinterpret_cast<const float4*>(turn + dim0));
                const double sn[2] = {w.x, w.z}, cs[2] = {w.y, w.w};
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const double x0 = x[2 * e], x1 = x[2 * e + 1];
                    x[2 * e] = __dsub_rn(__dmul_rn(x0, cs[e]), __dmul_rn(x1, sn[e]));
                    x[2 * e + 1] = __dadd_rn(__dmul_rn(x0, sn[e]), __dmul_rn(x1, cs[e]));
                }
            }
        }
        const double lo = -max8(fmax(fmax(-x[0], -x[1]), fmax(-x[2], -x[3]))), hi = max8(fmax(fmax(x[0], x[1]), fmax(x[2], x[3])));
        // fmax passes over NaN: whether a value of the block is one, or infinite, is asked for by itself
        const bool odd = !(fabs(x[0]) < 1e300 && fabs(x[1]) < 1e300 && fabs(x[2]) < 1e300 && fabs(x[3]) < 1e300);
        const bool bad = __ballot_sync(0xffffffffu, odd) >> (threadIdx.x & 24) & 0xff;
        const __half top = __ushort_as_half(0x7bff);
        __half m = __double2half(fmin(fmax(lo, -65504.0), 65504.0));
        const double mm = (double)__half2float(m);
        __half d = __double2half(fmin(fmax(hi - mm, 0.0) / 15.0, (double)__half2float(top)));
        if (bad) { m = __ushort_as_half(0x7fff); d = __ushort_as_half(0); }
        const double dd = (double)__half2float(d);
        uint32_t codes = 0;
        if (dd > 0.0) {
#pragma unroll
            for (int e = 0; e < 4; e++) codes |= (uint32_t)fmin(fmax(rint((x[e] - mm) / dd), 0.0), 15.0) << (4 * e);
        }
        if (p.in) {
            const CodePlace c = code_place(p, a.plan.tok_slot[p.tok], a.shape);
            *reinterpret_cast<uint16_t*>(a.pool + c.codes) = (uint16_t)codes;
            if (p.sub < 2) *reinterpret_cast<__half*>(a.pool + c.scales + p.sub * 2 * nb) = p.sub ? m : d;
        }
    }
}

__global__ void __launch_bounds__(256) kv4_read_kernel(const __grid_constant__ Kv4RowsArgs a) {
    pdl_launch_dependents();
    pdl_wait();
    const Kv4Head head = *a.plan.head;
    if (!kv4_fits(head, a.most_tokens, a.rope, a.shape, 0, a.status)) return;
    const uint32_t n = head.tokens, nb = a.shape.dim / KV4_BLOCK;
    const uint32_t lanes = n * a.shape.kv_heads * 2 * nb * 8;
    for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < lanes; i += gridDim.x * 256) {
        const RowPlace p = row_place(i, n, a.shape);
        const CodePlace c = code_place(p, a.plan.tok_slot[p.tok], a.shape);
        const uint32_t codes = __ldcg(reinterpret_cast<const unsigned short*>(a.pool + c.codes));
        const float d = f16_bits_to_f32(__ldcg(reinterpret_cast<const unsigned short*>(a.pool + c.scales)));
        const float m = f16_bits_to_f32(__ldcg(reinterpret_cast<const unsigned short*>(a.pool + c.scales + 2 * nb)));
        float4 o;      // d * code is exact in f32: one rounding
        o.x = __fmaf_rn(d, (float)(codes & 15), m);
        o.y = __fmaf_rn(d, (float)(codes >> 4 & 15), m);
        o.z = __fmaf_rn(d, (float)(codes >> 8 & 15), m);
        o.w = __fmaf_rn(d, (float)(codes >> 12), m);
        float* row = (p.value ? a.v + p.tok * a.v_ld : a.k + p.tok * a.k_ld) + (size_t)p.head * a.shape.dim;
        *reinterpret_cast<float4*>(row + p.block * KV4_BLOCK + p.sub * 4) = o;
    }
}

namespace {
template <class K>
cudaError_t launch_rows(K kernel, const Kv4RowsArgs& a, uint32_t tokens, int num_sms, cudaStream_t st, bool pdl) {
    if (!tokens) return cudaSuccess;
    cudaLaunchConfig_t lc = {}; cudaLaunchAttribute at[1];
    const size_t lanes = (size_t)tokens * a.shape.kv_heads * 2 * (a.shape.dim / KV4_BLOCK) * 8;
    const size_t ctas = (lanes + 255) / 256, most = (size_t)num_sms * 8;
    lc.gridDim = dim3((unsigned)(ctas < most ? ctas : most)); lc.blockDim = dim3(256); lc.stream = st;
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = at; lc.numAttrs = pdl ? 1 : 0;
    return cudaLaunchKernelEx(&lc, kernel, a);
}
}  // namespace

cudaError_t launch_kv4_append(const Kv4RowsArgs& a, uint32_t tokens, int num_sms, cudaStream_t st, bool pdl) { return launch_rows(kv4_append_kernel, a, tokens, num_sms, st, pdl); }
cudaError_t launch_kv4_read(const Kv4RowsArgs& a, uint32_t tokens, int num_sms, cudaStream_t st, bool pdl) { return launch_rows(kv4_read_kernel, a, tokens, num_sms, st, pdl); }

}  // namespace alice
