// Rows of keys and values into and out of the 4-bit cache (csrc/kv4.cuh).
#include <cuda_fp16.h>

#include "common.cuh"
#include "kv4.cuh"

namespace alice {

namespace {

// Four lanes hold one block of 32 values of one row, eight values each; a warp has eight blocks: two heads' rows of 128 dims, four of 64, one
// of 256. It takes the keys or the values of one token, `heads` key / value heads one after the other.
template <int NB>
struct Walk {
    static constexpr uint32_t DIM = 32 * NB, AT_ONCE = 8 / NB;      // heads a step takes
    uint32_t tok, head, end, dim0, pos;
    bool value;
    size_t codes, scales;        // of this lane's 8 codes (32 bits; of values 16 and, 2 NB further, 16), of its block's step (the minimum is 2 NB further), in the pool's head 0
    size_t per_head;
    __device__ __forceinline__ Walk(uint32_t unit, uint32_t heads, const Kv4Plan& plan, const Kv4Shape& s) {
        const uint32_t lane = threadIdx.x & 31, sub = lane & 3, chunks = (s.kv_heads + heads - 1) / heads, block = lane / 4 % NB;
        value = unit & 1;
        tok = (unit >> 1) / chunks;
        head = ((unit >> 1) - tok * chunks) * heads;
        end = min(head + heads, s.kv_heads);
        head += lane / 4 / NB;
        dim0 = block * KV4_BLOCK + sub * 8;
        const uint4 t = *reinterpret_cast<const uint4*>(plan.token + tok);
        pos = t.z;
        per_head = (size_t)s.tiles() * kv4_tile_bytes(DIM);
        const size_t tile = (size_t)t.x * kv4_tile_bytes(DIM);
        const uint32_t kr = kv4_row(t.y);
        codes = tile + (value ? kv4_v_codes(DIM) + t.y * (DIM / 2) + (2 * sub * NB + block) * 2 : kr * (DIM / 2) + kv4_k_word(NB, block, sub) * 4);
        scales = tile + (value ? kv4_v_scales(DIM) : kv4_k_scales(DIM)) + kr * (4 * NB) + block * 2;
    }
    static __host__ __device__ uint32_t units(uint32_t n, uint32_t heads, uint32_t kv_heads) { return n * ((kv_heads + heads - 1) / heads) * 2; }
};

template <class T>
__device__ __forceinline__ T min4(T v, uint32_t mask) {
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) v = min(v, __shfl_xor_sync(mask, v, o));
    return v;
}
template <class T>
__device__ __forceinline__ T max4(T v, uint32_t mask) {
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) v = max(v, __shfl_xor_sync(mask, v, o));
    return v;
}

struct Eight { float v[8]; };
__device__ __forceinline__ Eight load8(const float* p) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = reinterpret_cast<const float4*>(p)[1];
    return {{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
}
struct Held { uint32_t codes; __half d, m; };

// The formulas in f64, where products of f32 numbers are exact: x[e] = a[e] * cs[e] + b[e] * sn[e]. The four lanes of a block.
__device__ __forceinline__ Held held_exactly(const Eight& a, const Eight& b, const Eight& cs, const Eight& sn, uint32_t mask) {
    double x[8], lo = INFINITY, hi = -INFINITY;
    bool odd = false;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        x[e] = __dadd_rn(__dmul_rn((double)a.v[e], (double)cs.v[e]), __dmul_rn((double)b.v[e], (double)sn.v[e]));
        lo = fmin(lo, x[e]); hi = fmax(hi, x[e]);
        odd |= !(fabs(x[e]) < 1e300);      // minima and maxima pass over NaN: whether a value is one, or infinite, is asked for by itself
    }
    lo = min4(lo, mask); hi = max4(hi, mask);
    Held h;
    h.codes = 0;
    if (__any_sync(mask, odd)) {
        h.m = __ushort_as_half(0x7fff); h.d = __ushort_as_half(0);
        return h;
    }
    h.m = __double2half(fmin(fmax(lo, -65504.0), 65504.0));
    const double m = (double)__half2float(h.m);
    h.d = __double2half(fmin(fmax(hi - m, 0.0) / 15.0, 65504.0));
    const double d = (double)__half2float(h.d);
    if (d > 0.0) {
#pragma unroll
        for (int e = 0; e < 8; e++) h.codes |= (uint32_t)fmin(fmax(rint((x[e] - m) / d), 0.0), 15.0) << (4 * e);
    }
    return h;
}

// Minimum, step and codes in f32, together with how far f32 can be off; where that reaches over a border between two half-precision
// numbers or two codes (about one block in 300 of random keys, one in 700 of values), `border` says so.
// v = x cs + y sn is off by up to `off`, 0 for what is not rotated.
__device__ __forceinline__ Held held(const Eight& x, const Eight& y, const Eight& cs, const Eight& sn, bool turned, uint32_t mask, bool& border) {
    Eight v = x;
    float off = 0.0f;
    if (turned) {
        float far = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float s = y.v[e] * sn.v[e];
            v.v[e] = fmaf(x.v[e], cs.v[e], s);
            far = fmaxf(far, fabsf(x.v[e] * cs.v[e]) + fabsf(s));
        }
        // less than 2^-23 of the products' magnitudes (of all of the block), or 2^-149
        off = fmaf(max4(far, mask), 0x1p-22f, 0x1p-126f);
    }
    float lo = v.v[0], hi = v.v[0], all = fabsf(v.v[0]);
#pragma unroll
    for (int e = 1; e < 8; e++) { lo = fminf(lo, v.v[e]); hi = fmaxf(hi, v.v[e]); all += fabsf(v.v[e]); }
    lo = min4(lo, mask); hi = max4(hi, mask);
    // extremes within `off`: the same half at both ends? The step's: within a fifteenth of `off`, and 2^-21 of it (difference, factor and
    // product are off by less than 2^-22)
    const __half2 ms = __floats2half2_rn(lo - off, lo + off);
    const float m = __low2float(ms), step = fmaxf(hi - m, 0.0f) * (1.0f / 15.0f), slack = fmaf(step, 0x1p-21f, off * 0.07f);
    const __half2 ds = __floats2half2_rn(step - slack, step + slack);
    Held h;
    h.m = __low2half(ms); h.d = __low2half(ds);
    const float d = __low2float(ds), inv = __fdividef(1.0f, d);
    const uint32_t mb = *reinterpret_cast<const uint32_t*>(&ms), db = *reinterpret_cast<const uint32_t*>(&ds);
    // Numbers too large or steps too small for this, a NaN (which minima and maxima pass over, sums do not), an infinity; codes out of 0 .. 15
    border = (mb >> 16) != (mb & 0xffff) || (db >> 16) != (db & 0xffff) || !(d > 0x1p-20f) || !(all < 65000.0f) || !((lo - m) * inv > -0.45f && (hi - m) * inv < 15.45f);
    // a code is off by what v is, in steps, and less than 16 * 2^-21
    const float near = 0.5f - fmaf(off, inv, 0x1p-17f);
    float worst = 0;
    h.codes = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float c = (v.v[e] - m) * inv, r = c + 12582912.0f;      // 1.5 * 2^23: to the nearest whole number
        worst = fmaxf(worst, fabsf(c - (r - 12582912.0f)));
        h.codes |= (__float_as_uint(r) & 15u) << (4 * e);
    }
    border |= !(worst < near);
    return h;
}

}  // namespace

// Keys and values of a step into their pages. A warp's heads share the token's place and angles. 5470 tokens of 8 heads of 128 (52 MB read
// and written): 26.6 us, bound by latency: rows are asked for when those before are stored, for lack of registers (issue slots 54 %, 4.8 of the stalls an issue wait for
// loads); one head a warp takes 36, three CTAs an SM (80 registers) 30, all in f64 66.
template <int NB>
__global__ void __launch_bounds__(256, 4) kv4_append_kernel(const __grid_constant__ Kv4RowsArgs a) {
    using W = Walk<NB>;
    pdl_launch_dependents();
    pdl_wait();
    const Kv4Head all = *a.plan.head;
    if (!kv4_fits(all, a.most_tokens, a.rope, a.shape, a.status)) return;
    const uint32_t units = W::units(all.tokens, a.heads, a.shape.kv_heads), lane = threadIdx.x & 31, mask = 0xfu << (lane & 28);
    for (uint32_t u = blockIdx.x * 8 + (threadIdx.x >> 5); u < units; u += gridDim.x * 8) {
        W w(u, a.heads, a.plan, a.shape);
        const float* const row = w.value ? a.v + w.tok * a.v_ld : a.k + w.tok * a.k_ld;
        Eight cs{{1, 1, 1, 1, 1, 1, 1, 1}}, sn{{0, 0, 0, 0, 0, 0, 0, 0}};
        uint32_t other = w.dim0;
        if (!w.value && w.dim0 < a.rope.dims) {
            const float* const turn = a.rope.table + (size_t)(a.rope.by_token ? w.tok : w.pos) * a.rope.dims;
            const uint32_t half = a.rope.dims / 2;
            const bool upper = a.rope.neox && w.dim0 >= half;
            const uint32_t j = upper ? w.dim0 - half : w.dim0;
            const Eight t0 = load8(turn + (a.rope.neox ? 2 * j : w.dim0));
            if (a.rope.neox) {
                other = upper ? j : w.dim0 + half;
                const Eight t1 = load8(turn + 2 * j + 8);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float s = e < 4 ? t0.v[2 * e] : t1.v[2 * e - 8];
                    cs.v[e] = e < 4 ? t0.v[2 * e + 1] : t1.v[2 * e - 7];
                    sn.v[e] = upper ? s : -s;
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) { cs.v[e] = t0.v[e | 1]; sn.v[e] = e & 1 ? t0.v[e - 1] : -t0.v[e]; }
            }
        }
        // the whole warp one way or the other: what is not rotated loses nothing by cs = 1, sn = 0
        const bool turned = __any_sync(0xffffffffu, !w.value && w.dim0 < a.rope.dims);
        auto load = [&](uint32_t head, Eight& x, Eight& y) {
            const float* const at = row + (size_t)min(head, w.end - 1) * W::DIM;
            x = load8(at + w.dim0);
            if (turned && a.rope.neox) y = load8(at + other);
            else {
#pragma unroll
                for (int e = 0; e < 8; e++) y.v[e] = x.v[e ^ 1];
            }
        };
        auto store = [&](uint32_t head, const Held& h) {
            if (head >= w.end) return;
            uint8_t* const to = a.pool + w.codes + head * w.per_head;
            if (w.value) {
                *reinterpret_cast<uint16_t*>(to) = (uint16_t)h.codes;
                *reinterpret_cast<uint16_t*>(to + 2 * NB) = (uint16_t)(h.codes >> 16);
            } else *reinterpret_cast<uint32_t*>(to) = h.codes;
            if ((lane & 3) < 2) *reinterpret_cast<__half*>(a.pool + w.scales + head * w.per_head + (lane & 3) * 2 * NB) = lane & 3 ? h.m : h.d;
        };
        const uint32_t steps = (w.end - (w.head - lane / 4 / NB) + W::AT_ONCE - 1) / W::AT_ONCE;
        uint32_t again = 0;          // steps in which a block was near a border
        for (uint32_t i = 0; i < steps; i++) {
            Eight x, y;
            bool border;
            load(w.head + i * W::AT_ONCE, x, y);
            store(w.head + i * W::AT_ONCE, held(x, y, cs, sn, turned, mask, border));
            again |= __any_sync(0xffffffffu, border) ? 1u << i : 0u;
        }
        // those once more in f64, apart from the loop above, whose registers it would take
        for (; again; again &= again - 1) {
            const uint32_t head = w.head + (__ffs(again) - 1) * W::AT_ONCE;
            Eight x, y;
            load(head, x, y);
            store(head, held_exactly(x, y, cs, sn, mask));
        }
    }
}

// And out again: m + d * code, one rounding. 5470 tokens of 8 heads of 128 (45 MB of rows written, which stay in L2) 13.0 us, bound by latency: 7.4 stalls an issue wait for
// codes and scales of 2 and 4 bytes a lane, issue slots 51 %.
template <int NB>
__global__ void __launch_bounds__(256) kv4_read_kernel(const __grid_constant__ Kv4RowsArgs a) {
    using W = Walk<NB>;
    pdl_launch_dependents();
    pdl_wait();
    const Kv4Head all = *a.plan.head;
    if (!kv4_fits(all, a.most_tokens, a.rope, a.shape, a.status)) return;
    const uint32_t units = W::units(all.tokens, a.heads, a.shape.kv_heads);
    for (uint32_t u = blockIdx.x * 8 + (threadIdx.x >> 5); u < units; u += gridDim.x * 8) {
        W w(u, a.heads, a.plan, a.shape);
        float* const row = (w.value ? a.v + w.tok * a.v_ld : a.k + w.tok * a.k_ld) + w.dim0;
        for (; w.head < w.end; w.head += 4 * W::AT_ONCE) {
            uint32_t codes[4], dm[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {        // all loads ahead of the stores
                const uint8_t* const at = a.pool + min(w.head + i * W::AT_ONCE, w.end - 1) * w.per_head;
                codes[i] = w.value ? __ldcg(reinterpret_cast<const unsigned short*>(at + w.codes)) | (uint32_t)__ldcg(reinterpret_cast<const unsigned short*>(at + w.codes + 2 * NB)) << 16
                                   : __ldcg(reinterpret_cast<const unsigned int*>(at + w.codes));
                dm[i] = __ldcg(reinterpret_cast<const unsigned short*>(at + w.scales)) | (uint32_t)__ldcg(reinterpret_cast<const unsigned short*>(at + w.scales + 2 * NB)) << 16;
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float d = f16_bits_to_f32(dm[i] & 0xffff), m = f16_bits_to_f32(dm[i] >> 16);
                float o[8];      // d * code is exact in f32: one rounding
#pragma unroll
                for (int e = 0; e < 8; e++) o[e] = __fmaf_rn(d, __uint_as_float((codes[i] >> (4 * e) & 15u) | 0x4b000000u) - 8388608.0f, m);      // 2^23 + code, less 2^23
                // A pair of lanes stores its 16 values so that either store fills 32 bytes: halves of sectors took 17.6 us instead of 13.0.
                const bool odd = threadIdx.x & 1;
                float got[4];
#pragma unroll
                for (int e = 0; e < 4; e++) got[e] = __shfl_xor_sync(3u << (threadIdx.x & 30), odd ? o[e] : o[4 + e], 1);
                if (w.head + i * W::AT_ONCE < w.end) {
                    float* const to = row + (size_t)(w.head + i * W::AT_ONCE) * W::DIM;
                    *reinterpret_cast<float4*>(to - (odd ? 4 : 0)) = odd ? make_float4(got[0], got[1], got[2], got[3]) : make_float4(o[0], o[1], o[2], o[3]);
                    *reinterpret_cast<float4*>(to + (odd ? 4 : 8)) = odd ? make_float4(o[4], o[5], o[6], o[7]) : make_float4(got[0], got[1], got[2], got[3]);
                }
            }
        }
    }
}

// A model's one sequence: what the host works out for a batch (csrc/kv4_plan.cuh), from the position on the device.
__global__ void __launch_bounds__(256) kv4_plan_kernel(Kv4Plan plan, Kv4Shape s, uint32_t group, uint32_t rows, uint32_t n, const int* pos, uint32_t pos0, bool prompt) {
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t past = pos ? (uint32_t)*pos : pos0, total = n * group, jobs = (total + rows - 1) / rows, tid = threadIdx.x;
    auto tiles_of = [&](uint32_t j) { return (past + (min((j + 1) * rows, total) - 1) / group + 1 + KV4_TILE - 1) / KV4_TILE; };
    for (uint32_t i = tid; i < n; i += blockDim.x) {
        const uint32_t at = past + i;       // pages in order: page at / page_tokens
        const_cast<Kv4Token*>(plan.token)[i] = Kv4Token{at / s.page_tokens * s.kv_heads * s.tiles() + at % s.page_tokens / KV4_TILE, at % KV4_TILE, at, 0};
    }
    for (uint32_t j = tid; j < jobs; j += blockDim.x) {
        uint32_t before = 0;
        for (uint32_t i = 0; i < j; i++) before += tiles_of(i);
        const_cast<Kv4Job*>(plan.job)[prompt ? jobs - 1 - j : j] = Kv4Job{0, j * rows, min(rows, total - j * rows), 0, past, before, before + tiles_of(j), 0};
        const_cast<uint32_t*>(plan.job_tile)[j] = before;
        if (j == jobs - 1)
            *const_cast<Kv4Head*>(plan.head) = Kv4Head{1, n, prompt ? 0 : jobs, rows, prompt ? 0 : before + tiles_of(j), past + n, (past + n - 1) / s.page_tokens, prompt ? jobs : 0};
    }
}

cudaError_t launch_kv4_plan(const Kv4Plan& plan, const Kv4Shape& shape, uint32_t group, uint32_t n, const int* pos, uint32_t pos0, cudaStream_t st, bool pdl) {
    cudaLaunchConfig_t lc = {}; cudaLaunchAttribute at[1];
    lc.gridDim = dim3(1); lc.blockDim = dim3(256); lc.stream = st;
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = at; lc.numAttrs = pdl ? 1 : 0;
    const bool prompt = kv4_is_prompt(n * group, shape.dim);      // jobs that see most first
    return cudaLaunchKernelEx(&lc, kv4_plan_kernel, plan, shape, group, prompt ? KV4_PROMPT_ROWS : kv4_job_rows(n * group, shape.dim), n, pos, pos0, prompt);
}

namespace {
template <int NB, class K>
cudaError_t launch_rows(K kernel, Kv4RowsArgs a, uint32_t tokens, int num_sms, cudaStream_t st, bool pdl) {
    cudaLaunchConfig_t lc = {}; cudaLaunchAttribute at[1];
    // Heads a warp takes one after the other: as many as leave sixteen warps an SM. They share the token's place and angles, but a step of
    // few tokens wants its rows side by side.
    a.heads = Walk<NB>::AT_ONCE;
    while (a.heads < a.shape.kv_heads && a.heads < 8 && Walk<NB>::units(tokens, 2 * a.heads, a.shape.kv_heads) >= 16u * num_sms) a.heads *= 2;
    const uint32_t ctas = max((Walk<NB>::units(tokens, a.heads, a.shape.kv_heads) + 7) / 8, 1u), most = (uint32_t)num_sms * 32;
    lc.gridDim = dim3(ctas < most ? ctas : most); lc.blockDim = dim3(256); lc.stream = st;
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = at; lc.numAttrs = pdl ? 1 : 0;
    return cudaLaunchKernelEx(&lc, kernel, a);
}
}  // namespace

cudaError_t launch_kv4_append(const Kv4RowsArgs& a, uint32_t tokens, int num_sms, cudaStream_t st, bool pdl) {
    switch (a.shape.dim) {
        case 64: return launch_rows<2>(kv4_append_kernel<2>, a, tokens, num_sms, st, pdl);
        case 128: return launch_rows<4>(kv4_append_kernel<4>, a, tokens, num_sms, st, pdl);
        case 256: return launch_rows<8>(kv4_append_kernel<8>, a, tokens, num_sms, st, pdl);
        default: return cudaErrorInvalidValue;
    }
}
cudaError_t launch_kv4_read(const Kv4RowsArgs& a, uint32_t tokens, int num_sms, cudaStream_t st, bool pdl) {
    switch (a.shape.dim) {
        case 64: return launch_rows<2>(kv4_read_kernel<2>, a, tokens, num_sms, st, pdl);
        case 128: return launch_rows<4>(kv4_read_kernel<4>, a, tokens, num_sms, st, pdl);
        case 256: return launch_rows<8>(kv4_read_kernel<8>, a, tokens, num_sms, st, pdl);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace alice
