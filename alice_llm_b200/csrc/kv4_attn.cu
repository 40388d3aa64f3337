// Attention of one or several new tokens over the 4-bit cache (csrc/kv4.cuh).
//
// A warp takes a job's 4, 8 or 16 (token, query head) rows against tiles of 16 keys with m16n8k16 products in half precision:
//   scores^T [key][row]  = sum over blocks of d * (codes . q) + m * (sum of q)
//   out^T [dim][row]    += codes * (p * d), and m * p apart in f32
// with d, m a block's step and minimum. Codes enter less 8 (and m is m + 8 d), so that the two parts of a sum over many keys do not
// cancel; unpacking two of them is a mask and an exact addition in half precision. (Masked bits alone are exact operands too, as numbers
// below 2^-14, but the products of those lose bits in the sum: results were 4e-5 to 4e-4 off.) The other operand, q or p * d, is a pair of half-precision
// numbers (value and remainder, 22 bits), scaled by powers of two into the middle of their range.
// With up to 4 rows the pair fills two columns of the product, with more they are two products.
//
// All tiles of all jobs and key heads are one row of work that is cut into equal parts, a CTA an SM and again among its warps, so batches of any
// lengths are even. A warp streams its tiles through a ring of its own (cp.async); rows that several warps or CTAs had a part in are
// joined in shared memory, then by the CTA that is the last to bring its part.
//
// The running maximum m only moves when a score exceeds it by 2^8, and weighted sums go to f32 sums every 16 tiles: products
// on tensor cores add up with less than f32 rounding, which over a long chain would add up itself.
#include <cuda_fp16.h>

#include "common.cuh"
#include "kv4.cuh"

namespace alice {

namespace {

constexpr int STAGES = 3;
constexpr uint32_t FLUSH = 16;       // tiles
constexpr uint32_t MAX_CTAS = 192;
constexpr float ROOM = 8.0f;         // what a score may exceed the reference by, in powers of two

template <int NB, int R>
struct Cfg {
    static constexpr bool SPLIT = R == 4;
    static constexpr int NT = R == 16 ? 2 : 1;                    // eight-column products
    static constexpr int RT = SPLIT ? 1 : 2 * NT;                 // rows a lane has scores and outputs of
    static constexpr int WARPS = NB == 8 ? (R == 4 ? 8 : 6) : R == 4 ? 16 : R == 8 ? 12 : 8;
    static constexpr uint32_t DIM = 32 * NB, TILE = kv4_tile_bytes(DIM);
    static constexpr int NF = NB * RT;                            // float4 of output a lane has
    static constexpr uint32_t PART = R * DIM + 2 * R;             // floats of a part of a job
    struct Smem {
        float4 sum[WARPS][2][NF][32];
        float2 ml[WARPS][2][R];                                   // reference and sum of weights
        long long seg_job[WARPS][2];                              // key head * jobs + job, -1: nothing to join
        uint32_t seg_ends[WARPS][2];                              // 1: has the job's first tile, 2: its last
        float weight[2 * WARPS][R], total[R];
        uint32_t last[2];
        alignas(16) uint8_t ring[WARPS][STAGES][TILE];
    };
};

__device__ __forceinline__ uint32_t half2_bits(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }
__device__ __forceinline__ __half2 bits_half2(uint32_t u) { return *reinterpret_cast<const __half2*>(&u); }
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the same with a sum that starts at zero
__device__ __forceinline__ void mma_f16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
// The eight codes of a word less 8, two to a register: .. [0] nibbles 0 and 4, [1] 1 and 5, [2] 2 and 6, [3] 3 and 7. Four bits put under
// the exponent of 1024 are 1024 + code, or with the next four 1024 + 16 code; both steps are exact.
struct Codes { uint32_t v[4]; };
__device__ __forceinline__ Codes unpack(uint32_t x) {
    constexpr uint32_t MAGIC = 0x64006400u, EVEN = 0x000f000fu, ODD = 0x00f000f0u;
    const __half2 less = __half2half2(__ushort_as_half(0xe408)), sixteenth = __half2half2(__ushort_as_half(0x2c00)), less16 = __half2half2(__ushort_as_half(0xd480));  // -1032, 1 / 16, -72
    const uint32_t y = x >> 8;
    Codes c;
    c.v[0] = half2_bits(__hadd2(bits_half2(x & EVEN | MAGIC), less));
    c.v[1] = half2_bits(__hfma2(bits_half2(x & ODD | MAGIC), sixteenth, less16));
    c.v[2] = half2_bits(__hadd2(bits_half2(y & EVEN | MAGIC), less));
    c.v[3] = half2_bits(__hfma2(bits_half2(y & ODD | MAGIC), sixteenth, less16));
    return c;
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }    // -126 <= e <= 127
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }

// Words of a row that a lane reads in one go.
template <int N>
struct Words { uint32_t w[N]; };
template <int N>
__device__ __forceinline__ Words<N> lds_words(uint32_t a) {
    Words<N> r;
    if constexpr (N == 1) r.w[0] = lds32(a);
    else if constexpr (N == 2) { const uint2 v = lds64(a); r.w[0] = v.x; r.w[1] = v.y; }
    else {
#pragma unroll
        for (int i = 0; i < N / 4; i++) { const uint4 v = lds128(a + 16 * i); r.w[4 * i] = v.x; r.w[4 * i + 1] = v.y; r.w[4 * i + 2] = v.z; r.w[4 * i + 3] = v.w; }
    }
    return r;
}

// 8 consecutive floats of a query, from dim0 on, rotated.
__device__ __forceinline__ void rotated8(float (&x)[8], const float* q, uint32_t dim0, const float* turn, const Kv4Rope& rope) {
    auto load8 = [](float (&v)[8], const float* p) {
        const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    };
    load8(x, q + dim0);
    if (dim0 >= rope.dims) return;
    if (rope.neox) {
        const uint32_t half = rope.dims / 2;
        const bool upper = dim0 >= half;
        const uint32_t j = upper ? dim0 - half : dim0;
        float other[8], w0[8], w1[8];
        load8(other, q + (upper ? j : dim0 + half));
        load8(w0, turn + 2 * j);
        load8(w1, turn + 2 * j + 8);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float sn = e < 4 ? w0[2 * e] : w1[2 * e - 8], cs = e < 4 ? w0[2 * e + 1] : w1[2 * e - 7];
            x[e] = x[e] * cs + (upper ? other[e] * sn : -(other[e] * sn));
        }
    } else {
        float w[8];
        load8(w, turn + dim0);
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const float a = x[e], b = x[e + 1];
            x[e] = a * w[e + 1] - b * w[e];
            x[e + 1] = a * w[e] + b * w[e + 1];
        }
    }
}

// The job that tile x of a key head belongs to: the last with job_tile <= x. All lanes look, 32 places at a time.
__device__ __forceinline__ uint32_t find_job(const uint32_t* job_tile, uint32_t jobs, uint32_t x, uint32_t lane) {
    uint32_t lo = 0, n = jobs;
    while (n > 1) {
        const uint32_t step = (n + 31) / 32, i = lo + lane * step;
        const uint32_t hit = __ballot_sync(0xffffffffu, lane * step < n && __ldg(job_tile + i) <= x);
        const uint32_t k = 31 - __clz(hit);
        n = min(step, n - k * step);
        lo += k * step;
    }
    return lo;
}

struct Job {
    uint32_t seq, row, rows, first, past, tile0, tile1;   // row: of the sequence's (token, head) rows; rows: how many it has from there
};
__device__ __forceinline__ Job get_job(const Kv4Plan& p, uint32_t j, uint32_t group, uint32_t most) {
    Job b;
    b.seq = __ldg(p.job_seq + j); b.row = __ldg(p.job_row + j); b.tile0 = __ldg(p.job_tile + j); b.tile1 = __ldg(p.job_tile + j + 1);
    b.first = __ldg(p.seq_first + b.seq); b.past = __ldg(p.seq_past + b.seq);
    b.rows = min(most, __ldg(p.seq_count + b.seq) * group - b.row);
    return b;
}

}  // namespace

template <int NB, int R>
__global__ void __launch_bounds__(Cfg<NB, R>::WARPS * 32, 1) kv4_attn_kernel(const __grid_constant__ Kv4AttnArgs a) {
    using C = Cfg<NB, R>;
    constexpr int NT = C::NT, RT = C::RT, NF = C::NF, W = C::WARPS;
    constexpr bool SPLIT = C::SPLIT;
    constexpr uint32_t DIM = C::DIM, TILE = C::TILE;
    extern __shared__ __align__(16) uint8_t raw[];
    auto& sh = *reinterpret_cast<typename C::Smem*>(raw);
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    pdl_launch_dependents();
    pdl_wait();
    const Kv4Plan& pl = a.plan;
    const Kv4Head hd = *pl.head;
    if (!kv4_fits(hd, a.most_tokens, a.rope, a.shape, R, a.status)) return;
    const unsigned long long total = (unsigned long long)hd.tiles * a.shape.kv_heads;
    // a part of a CTA is at least a tile for each of its warps
    const uint32_t grid = (uint32_t)min((unsigned long long)gridDim.x, (total + W - 1) / W);
    if (blockIdx.x >= grid) return;
    const unsigned long long c0 = total * blockIdx.x / grid, c1 = total * (blockIdx.x + 1) / grid;
    const unsigned long long w0 = c0 + (c1 - c0) * warp / W, w1 = c0 + (c1 - c0) * (warp + 1) / W;
    if (lane < 2) sh.seg_job[warp][lane] = -1;

    if (w0 < w1) {
        // ---- the ring: tiles are asked for STAGES - 1 ahead ----
        const uint32_t ring = smem_u32(sh.ring[warp][0]);
        const uint32_t per_page = a.shape.tiles();
        uint32_t p_head = (uint32_t)(w0 / hd.tiles), p_tile = (uint32_t)(w0 - (unsigned long long)p_head * hd.tiles);
        uint32_t p_job = find_job(pl.job_tile, hd.jobs, p_tile, lane);
        uint32_t job = p_job, head = p_head;
        uint32_t p_seq = 0, p_tile0 = 0, p_end = 0, p_pages = 0, p_base = 0xffffffffu;    // of the job; pages of 32 pages, a lane each
        uint32_t p_left = 0;                                                             // tiles to come of the page and the job
        const uint8_t* p_src = nullptr;
        uint32_t p_count = (uint32_t)(w1 - w0);
        bool p_new = true;
        auto ask = [&](uint32_t stage) {
            if (p_count) {
                p_count--;
                if (p_left == 0) {
                    if (p_new) {
                        p_seq = __ldg(pl.job_seq + p_job); p_tile0 = __ldg(pl.job_tile + p_job); p_end = __ldg(pl.job_tile + p_job + 1);
                        p_base = 0xffffffffu; p_new = false;
                    }
                    const uint32_t i = p_tile - p_tile0, n = i / per_page, in = i - n * per_page;
                    if (p_base == 0xffffffffu || n >= p_base + 32) {
                        p_base = n;
                        p_pages = __ldg(pl.table + (size_t)p_seq * pl.table_ld + min(n + lane, (p_end - 1 - p_tile0) / per_page));
                    }
                    const uint32_t page = __shfl_sync(0xffffffffu, p_pages, n - p_base);
                    p_src = a.pool + (((size_t)page * a.shape.kv_heads + p_head) * per_page + in) * TILE + lane * 16;
                    p_left = min(per_page - in, p_end - p_tile);
                }
                const uint32_t dst = ring + stage * TILE + lane * 16;
#pragma unroll
                for (uint32_t c = 0; c < (TILE / 16 + 31) / 32; c++)
                    if (TILE % 512 == 0 || c * 512 + lane * 16 < TILE) cp16(dst + c * 512, p_src + c * 512);
                p_src += TILE; p_tile++;
                if (--p_left == 0 && p_tile == p_end) {
                    p_new = true; p_job++;
                    if (p_tile == hd.tiles) { p_tile = 0; p_job = 0; p_head++; }
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int s = 0; s < STAGES - 1; s++) ask(s);

        uint32_t stage = 0, slot = 0;
        for (unsigned long long at = w0; at < w1;) {
            // ---- a job, or this warp's part of it ----
            const Job jb = get_job(pl, job, a.group, R);
            const unsigned long long j0 = (unsigned long long)head * hd.tiles + jb.tile0, j1 = (unsigned long long)head * hd.tiles + jb.tile1;
            const unsigned long long end = min(j1, w1);
            const bool has_first = at == j0, has_last = end == j1;

            // queries: columns of the product in the order of a lane's codes, and what each row needs beside them
            uint32_t qf[NT][NB][SPLIT ? 4 : 8];      // [..][0..3]: (value, or by column value and remainder), [4..7]: remainders
            float qsum[RT][NB], factor[RT];
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const uint32_t row = SPLIT ? g >> 1 : n * 8 + g;
                const bool there = row < jb.rows;
                const uint32_t r = jb.row + (there ? row : 0), tok = r / a.group, qh = head * a.group + r % a.group, at_tok = jb.first + tok;
                const float* q = a.q + at_tok * a.q_ld + (size_t)qh * DIM;
                const float* turn = a.rope.table + (size_t)(a.rope.by_token ? at_tok : jb.past + tok) * a.rope.dims;
                float x[NB][8], top = 0;
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    rotated8(x[b], q, b * 32 + 8 * t, turn, a.rope);
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        x[b][e] = there ? x[b][e] * a.scale : 0.0f;      // log2(e) comes with the factor below: a lone rounding of the score
                        top = fmaxf(top, fabsf(x[b][e]));
                    }
                }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                int e2 = (int)((__float_as_uint(top) >> 23) & 0xff) - 127 - 9;     // the largest into 2^9 .. 2^10
                e2 = min(max(e2, -100), 120);
                const float down = pow2(-e2);
                const float up = pow2(e2);
                const bool low = SPLIT && (g & 1);
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    float sum = 0;
#pragma unroll
                    for (int e = 0; e < 8; e++) sum += x[b][e] * down;
                    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float v0 = x[b][e] * down, v1 = x[b][e + 4] * down;
                        const __half2 hi = __floats2half2_rn(v0, v1);
                        const float2 back = __half22float2(hi);
                        const __half2 lo = __floats2half2_rn(v0 - back.x, v1 - back.y);
                        if (SPLIT) qf[n][b][e] = half2_bits(low ? lo : hi);
                        else { qf[n][b][e] = half2_bits(hi); qf[n][b][SPLIT ? 0 : 4 + e] = half2_bits(lo); }
                    }
                    if (SPLIT) qsum[0][b] = __shfl_sync(0xffffffffu, sum, t * 8);
                    else {
                        qsum[2 * n % RT][b] = __shfl_sync(0xffffffffu, sum, t * 8);
                        qsum[(2 * n + 1) % RT][b] = __shfl_sync(0xffffffffu, sum, t * 8 + 4);
                    }
                }
                const float f = up;
                if (SPLIT) factor[0] = __shfl_sync(0xffffffffu, f, t * 8) * 1.44269504088896341f;
                else {
                    factor[2 * n % RT] = __shfl_sync(0xffffffffu, f, t * 8) * 1.44269504088896341f;
                    factor[(2 * n + 1) % RT] = __shfl_sync(0xffffffffu, f, t * 8 + 4) * 1.44269504088896341f;
                }
            }
            uint32_t limit[RT], least = 0xffffffffu;        // positions a row sees
#pragma unroll
            for (int i = 0; i < RT; i++) {
                const uint32_t row = SPLIT ? t : (i >> 1) * 8 + 2 * t + (i & 1);
                limit[i] = row < jb.rows ? jb.past + (jb.row + row) / a.group + 1 : 0u;
                if (row < jb.rows) least = min(least, limit[i]);
            }
            least = __reduce_min_sync(0xffffffffu, least);

            float acc[NT][NB][2][4], accm[RT][NB], l[RT], ref[RT], lsum[RT], mref[RT];
#pragma unroll
            for (int i = 0; i < RT; i++) {
                l[i] = lsum[i] = 0; ref[i] = mref[i] = -INFINITY;
#pragma unroll
                for (int b = 0; b < NB; b++) accm[i][b] = 0;
            }
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int u = 0; u < 2; u++)
#pragma unroll
                        for (int c = 0; c < 4; c++) acc[n][b][u][c] = 0;
            uint32_t dtop = 0;                  // exponent field of the largest step so far, in the top bits of a half
            float dscale = 0, dback = 0;        // 2^z on p * d, and 2^-z
            uint32_t held = 0;                  // tiles in acc
            bool begun = false;                 // sums are in shared memory
            float4* const mine = &sh.sum[warp][slot][0][lane];

            // what acc, accm and l hold joins the sums in shared memory
            auto flush = [&]() {
#pragma unroll
                for (int i = 0; i < RT; i++) {
                    const float c = mref[i] == ref[i] ? 1.0f : ex2(mref[i] - ref[i]);
                    float s = l[i];
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
                    lsum[i] = begun ? lsum[i] * c + s : s;
                    l[i] = 0; mref[i] = ref[i];
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        float am = accm[i][b];
#pragma unroll
                        for (int o = 4; o < 32; o <<= 1) am += __shfl_xor_sync(0xffffffffu, am, o);
                        accm[i][b] = 0;
                        float v[4];
#pragma unroll
                        for (int u = 0; u < 2; u++) {
                            float (&x)[4] = acc[SPLIT ? 0 : i >> 1][b][u];
                            if (SPLIT) { v[2 * u] = x[0] + x[1]; v[2 * u + 1] = x[2] + x[3]; x[0] = x[1] = x[2] = x[3] = 0; }
                            else { v[2 * u] = x[i & 1]; v[2 * u + 1] = x[2 + (i & 1)]; x[i & 1] = x[2 + (i & 1)] = 0; }
                        }
                        float4 o = make_float4(fmaf(v[0], dback, am), fmaf(v[1], dback, am), fmaf(v[2], dback, am), fmaf(v[3], dback, am));
                        float4* to = mine + (i * NB + b) * 32;
                        if (begun) { const float4 p = *to; o.x = fmaf(p.x, c, o.x); o.y = fmaf(p.y, c, o.y); o.z = fmaf(p.z, c, o.z); o.w = fmaf(p.w, c, o.w); }
                        *to = o;
                    }
                }
                held = 0; begun = true;
            };

            uint32_t key0 = (uint32_t)(at - j0) * KV4_TILE;
            for (; at < end; at++, key0 += KV4_TILE) {
                asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
                __syncwarp();
                ask((stage + STAGES - 1) % STAGES);       // where the tile before this one was: every lane is done with it
                const uint32_t base = ring + stage * TILE;
                // ---- scores ----
                float s[RT][2];                 // of keys tau(g), 8 + tau(g)
#pragma unroll
                for (int i = 0; i < RT; i++) s[i][0] = s[i][1] = 0;
                const uint32_t krow = base + g * (DIM / 2), srow = base + kv4_k_scales(DIM) + g * (4 * NB);
#pragma unroll
                for (int h = 0; h < (NB + 3) / 4; h++) {
                    constexpr int NW = NB < 4 ? NB : 4;
                    const uint32_t kat = krow + (NB == 8 ? h * 64 + t * 16 : t * NB * 4);
                    const Words<NW> ka = lds_words<NW>(kat), kb = lds_words<NW>(kat + 4 * DIM);
                    const Words<NW> sa = lds_words<NW>(srow + h * 16), sb = lds_words<NW>(srow + h * 16 + 32 * NB);
#pragma unroll
                    for (int w = 0; w < NW; w++) {
                        const int b = h * 4 + w;
                        const Codes xa = unpack(ka.w[w]), xb = unpack(kb.w[w]);
                        float2 da = __half22float2(bits_half2(sa.w[w])), db = __half22float2(bits_half2(sb.w[w]));
                        da.y = fmaf(8.0f, da.x, da.y); db.y = fmaf(8.0f, db.x, db.y);       // what a code of 8 stands for
#pragma unroll
                        for (int n = 0; n < NT; n++) {
                            float c[4];
                            mma_f16_first(c, xa.v[0], xb.v[0], xa.v[1], xb.v[1], qf[n][b][0], qf[n][b][1]);
                            mma_f16(c, xa.v[2], xb.v[2], xa.v[3], xb.v[3], qf[n][b][2], qf[n][b][3]);
                            if (!SPLIT) {
                                mma_f16(c, xa.v[0], xb.v[0], xa.v[1], xb.v[1], qf[n][b][SPLIT ? 0 : 4], qf[n][b][SPLIT ? 0 : 5]);
                                mma_f16(c, xa.v[2], xb.v[2], xa.v[3], xb.v[3], qf[n][b][SPLIT ? 0 : 6], qf[n][b][SPLIT ? 0 : 7]);
                            }
                            if (SPLIT) {
                                s[0][0] = fmaf(da.x, c[0] + c[1], fmaf(da.y, qsum[0][b], s[0][0]));
                                s[0][1] = fmaf(db.x, c[2] + c[3], fmaf(db.y, qsum[0][b], s[0][1]));
                            } else {
#pragma unroll
                                for (int j = 0; j < 2; j++) {
                                    const int i = (2 * n + j) % RT;
                                    s[i][0] = fmaf(da.x, c[j], fmaf(da.y, qsum[i][b], s[i][0]));
                                    s[i][1] = fmaf(db.x, c[2 + j], fmaf(db.y, qsum[i][b], s[i][1]));
                                }
                            }
                        }
                    }
                }
                // ---- weights ----
                const uint32_t tau = (g >> 1) + 4 * (g & 1), keyA = key0 + tau, keyB = keyA + 8;
                const uint32_t vsrow = base + kv4_v_scales(DIM) + g * (4 * NB);
                Words<NB> va = lds_words<NB>(vsrow), vb = lds_words<NB>(vsrow + 32 * NB);
                const bool edge = key0 + KV4_TILE > least;       // some row does not see all of the tile
                bool move = false;
#pragma unroll
                for (int i = 0; i < RT; i++) {
                    s[i][0] *= factor[i]; s[i][1] *= factor[i];
                    if (edge) {
                        if (keyA >= limit[i]) s[i][0] = -INFINITY;
                        if (keyB >= limit[i]) s[i][1] = -INFINITY;
                    }
                    move |= fmaxf(s[i][0], s[i][1]) > ref[i] + ROOM;
                }
                if (edge) {      // keys that no row sees: whatever lies there has no part
                    uint32_t far = limit[0];
#pragma unroll
                    for (int i = 1; i < RT; i++) far = max(far, limit[i]);
                    far = __reduce_max_sync(0xffffffffu, far);
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        if (keyA >= far) va.w[b] = 0;
                        if (keyB >= far) vb.w[b] = 0;
                    }
                }
                __half2 both = __hmax2(bits_half2(va.w[0]), bits_half2(vb.w[0]));
#pragma unroll
                for (int b = 1; b < NB; b++) both = __hmax2(both, __hmax2(bits_half2(va.w[b]), bits_half2(vb.w[b])));
                const uint32_t dmax = half2_bits(both) & 0x7c00u;
                move |= dmax > dtop;
                if (__any_sync(0xffffffffu, move)) {
                    if (held) flush();
                    dtop = __reduce_max_sync(0xffffffffu, max(dmax, dtop));
                    // steps below 2^(e + 1), weights up to 2^8: their products into less than 2^15
                    const int z = 6 - ((int)(dtop >> 10) - 15);
                    dscale = pow2(z); dback = pow2(-z);
#pragma unroll
                    for (int i = 0; i < RT; i++) {
                        float m = fmaxf(s[i][0], s[i][1]);
#pragma unroll
                        for (int o = 4; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                        ref[i] = fmaxf(ref[i], m);
                    }
                }
                float p[RT][2];
#pragma unroll
                for (int i = 0; i < RT; i++) {
                    p[i][0] = ex2(s[i][0] - ref[i]); p[i][1] = ex2(s[i][1] - ref[i]);
                    if (edge) {
                        if (keyA >= limit[i]) p[i][0] = 0;
                        if (keyB >= limit[i]) p[i][1] = 0;
                    }
                    l[i] += p[i][0] + p[i][1];
                }
                // ---- values ----
                Words<(NB + 1) / 2> v[4];
                const uint32_t vrow = base + kv4_v_codes(DIM) + t * (DIM / 2) + g * (2 * NB);
#pragma unroll
                for (int i = 0; i < 4; i++) v[i] = lds_words<(NB + 1) / 2>(vrow + i * 2 * DIM);
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    const uint32_t pick = b & 1 ? 0x7632u : 0x5410u;
                    const uint32_t xa = __byte_perm(v[0].w[b / 2], v[1].w[b / 2], pick), xb = __byte_perm(v[2].w[b / 2], v[3].w[b / 2], pick);
                    const Codes ca = unpack(xa), cb = unpack(xb);
                    const float dax = __low2float(bits_half2(va.w[b])) * dscale, dbx = __low2float(bits_half2(vb.w[b])) * dscale;
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        if (SPLIT) {
                            const float wa = p[0][0] * dax, wb = p[0][1] * dbx;
                            const __half ha = __float2half_rn(wa), hb = __float2half_rn(wb);
                            const uint32_t b0 = transposed(half2_bits(__halves2half2(ha, __float2half_rn(wa - __half2float(ha)))));
                            const uint32_t b1 = transposed(half2_bits(__halves2half2(hb, __float2half_rn(wb - __half2float(hb)))));
                            mma_f16(acc[0][b][0], ca.v[0], ca.v[1], cb.v[0], cb.v[1], b0, b1);
                            mma_f16(acc[0][b][1], ca.v[2], ca.v[3], cb.v[2], cb.v[3], b0, b1);
                        } else {
                            const int i = 2 * n % RT, j = (2 * n + 1) % RT;
                            const float a0 = p[i][0] * dax, a1 = p[j][0] * dax, e0 = p[i][1] * dbx, e1 = p[j][1] * dbx;
                            const __half2 ha = __floats2half2_rn(a0, a1), hb = __floats2half2_rn(e0, e1);
                            const float2 fa = __half22float2(ha), fb = __half22float2(hb);
                            const uint32_t b0 = transposed(half2_bits(ha)), b1 = transposed(half2_bits(hb));
                            const uint32_t d0 = transposed(half2_bits(__floats2half2_rn(a0 - fa.x, a1 - fa.y))), d1 = transposed(half2_bits(__floats2half2_rn(e0 - fb.x, e1 - fb.y)));
                            mma_f16(acc[n][b][0], ca.v[0], ca.v[1], cb.v[0], cb.v[1], b0, b1);
                            mma_f16(acc[n][b][1], ca.v[2], ca.v[3], cb.v[2], cb.v[3], b0, b1);
                            mma_f16(acc[n][b][0], ca.v[0], ca.v[1], cb.v[0], cb.v[1], d0, d1);
                            mma_f16(acc[n][b][1], ca.v[2], ca.v[3], cb.v[2], cb.v[3], d0, d1);
                        }
                    }
                }
                // minima: of a key that a row does not see not even a NaN
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    float2 da = __half22float2(bits_half2(va.w[b])), db = __half22float2(bits_half2(vb.w[b]));
                    const float ma = fmaf(8.0f, da.x, da.y), mb = fmaf(8.0f, db.x, db.y);
#pragma unroll
                    for (int i = 0; i < RT; i++) {
                        if (!edge) accm[i][b] = fmaf(p[i][0], ma, fmaf(p[i][1], mb, accm[i][b]));
                        else {
                            if (keyA < limit[i]) accm[i][b] = fmaf(p[i][0], ma, accm[i][b]);
                            if (keyB < limit[i]) accm[i][b] = fmaf(p[i][1], mb, accm[i][b]);
                        }
                    }
                }
                held++;
                stage = stage + 1 == STAGES ? 0 : stage + 1;
                if (held == FLUSH) flush();
            }
            if (held) flush();

            if (has_first && has_last) {        // all of the job: out it goes
#pragma unroll
                for (int i = 0; i < RT; i++) {
                    const uint32_t row = SPLIT ? t : (i >> 1) * 8 + 2 * t + (i & 1);
                    if (row < jb.rows) {
                        const uint32_t r = jb.row + row;
                        float* out = a.out + (size_t)(jb.first + r / a.group) * a.out_ld + (size_t)(head * a.group + r % a.group) * DIM + 4 * g;
                        const float inv = 1.0f / lsum[i];
#pragma unroll
                        for (int b = 0; b < NB; b++) {
                            const float4 o = mine[(i * NB + b) * 32];
                            *reinterpret_cast<float4*>(out + b * 32) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
                        }
                    }
                }
            } else {
                if (g == 0) {
#pragma unroll
                    for (int i = 0; i < RT; i++) sh.ml[warp][slot][SPLIT ? t : (i >> 1) * 8 + 2 * t + (i & 1)] = make_float2(mref[i], lsum[i]);
                }
                if (lane == 0) {
                    sh.seg_job[warp][slot] = (long long)head * hd.jobs + job;
                    sh.seg_ends[warp][slot] = (has_first ? 1u : 0u) | (has_last ? 2u : 0u);
                }
            }
            slot = 1;
            if (has_last) {
                job++;
                if (job == hd.jobs) { job = 0; head++; }
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    }

    // ---- parts of jobs: joined in the CTA, then by the last CTA of each job ----
    if (tid < 2) sh.last[tid] = 0;
    __syncthreads();
    const long long my_job = lane < 2 * W ? sh.seg_job[lane >> 1][lane & 1] : -1;
    const uint32_t my_ends = my_job >= 0 ? sh.seg_ends[lane >> 1][lane & 1] : 0u;
    const uint32_t valid = __ballot_sync(0xffffffffu, my_job >= 0);
    // a row's place in the fragments: element f = (i * NB + b) * 32 + lane
    auto row_of = [](uint32_t f) { const uint32_t i = f / (NB * 32), ln = f & 31; return SPLIT ? ln & 3 : (i >> 1) * 8 + 2 * (ln & 3) + (i & 1); };
    auto store_out = [&](long long jid, uint32_t f, float4 o, float l) {
        const uint32_t head = (uint32_t)(jid / hd.jobs);
        const Job jb = get_job(pl, (uint32_t)(jid - (long long)head * hd.jobs), a.group, R);
        const uint32_t row = row_of(f);
        if (row >= jb.rows) return;
        const uint32_t r = jb.row + row, b = f / 32 % NB, ln = f & 31;
        const float inv = 1.0f / l;
        float* out = a.out + (size_t)(jb.first + r / a.group) * a.out_ld + (size_t)(head * a.group + r % a.group) * DIM + b * 32 + 4 * (ln >> 2);
        *reinterpret_cast<float4*>(out) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    };
    auto part_at = [&](uint32_t cta, uint32_t which) { return a.part + ((size_t)cta * 2 + which) * C::PART; };
    // weights of the parts: a warp a row, a part a lane
    for (uint32_t row = warp; row < R; row += W) {
        float2 ml = my_job >= 0 ? sh.ml[lane >> 1][lane & 1][row] : make_float2(0, 0);
        for (uint32_t left = valid; left;) {
            const long long jid = __shfl_sync(0xffffffffu, my_job, __ffs(left) - 1);
            const bool member = my_job == jid;
            left &= ~__ballot_sync(0xffffffffu, member);
            float m = member ? ml.x : -INFINITY;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            const float c = member ? ml.x == m ? 1.0f : ex2(ml.x - m) : 0.0f;
            float l = member ? ml.y * c : 0.0f;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
            if (member) { sh.ml[lane >> 1][lane & 1][row] = make_float2(m, l); sh.weight[lane][row] = c; }
        }
    }
    __syncthreads();
    long long open_job[2] = {-1, -1};        // of this CTA: one that began before it, one that began in it
    for (uint32_t left = valid; left;) {
        const int first = __ffs(left) - 1;
        const long long jid = __shfl_sync(0xffffffffu, my_job, first);
        const uint32_t members = __ballot_sync(0xffffffffu, my_job == jid);
        const uint32_t ends = __reduce_or_sync(0xffffffffu, my_job == jid ? my_ends : 0u);
        left &= ~members;
        if (ends == 1) open_job[1] = jid;
        if (!(ends & 1)) open_job[0] = jid;
        for (uint32_t f = tid; f < NF * 32; f += W * 32) {
            const uint32_t row = row_of(f);
            float4 o = make_float4(0, 0, 0, 0);
#pragma unroll 4
            for (uint32_t e = first; e < 2 * W; e++) {
                if (!(members >> e & 1)) continue;
                const float c = sh.weight[e][row];
                const float4 x = (&sh.sum[e >> 1][e & 1][0][0])[f];
                o.x = fmaf(x.x, c, o.x); o.y = fmaf(x.y, c, o.y); o.z = fmaf(x.z, c, o.z); o.w = fmaf(x.w, c, o.w);
            }
            const float2 ml = sh.ml[first >> 1][first & 1][row];
            if (ends == 3) store_out(jid, f, o, ml.y);
            else {
                float* to = part_at(blockIdx.x, ends & 1);
                __stcg(reinterpret_cast<float4*>(to) + f, o);
                if ((f / 32) % NB == 0 && (f & 31) < 4) __stcg(reinterpret_cast<float2*>(to + R * DIM) + row, ml);
            }
        }
    }
    if (open_job[0] < 0 && open_job[1] < 0) return;
    __threadfence();
    __syncthreads();
    uint32_t first_cta[2], count[2];
#pragma unroll
    for (int k = 0; k < 2; k++) {
        first_cta[k] = count[k] = 0;
        if (open_job[k] < 0) continue;
        const unsigned long long head = open_job[k] / hd.jobs, j = open_job[k] - head * hd.jobs;
        const unsigned long long j0 = head * hd.tiles + __ldg(pl.job_tile + j), j1 = head * hd.tiles + __ldg(pl.job_tile + j + 1);
        first_cta[k] = (uint32_t)(((j0 + 1) * grid - 1) / total);
        count[k] = (uint32_t)((j1 * grid - 1) / total) - first_cta[k] + 1;
        if (tid == 0 && atomicAdd(a.tickets + first_cta[k], 1u) == count[k] - 1) {
            a.tickets[first_cta[k]] = 0;
            sh.last[k] = 1;
        }
    }
    __syncthreads();
#pragma unroll 1
    for (int k = 0; k < 2; k++) {
        if (!sh.last[k]) continue;
        __threadfence();
        // weights of the CTAs' parts, where the ring was
        float2* const ml = reinterpret_cast<float2*>(sh.ring[0][0]);
        static_assert(sizeof(sh.ring) >= sizeof(float2) * R * MAX_CTAS, "a weight a row of every CTA");
        for (uint32_t i = tid; i < count[k] * R; i += W * 32)
            ml[i] = __ldcg(reinterpret_cast<const float2*>(part_at(first_cta[k] + i / R, i < R) + R * DIM) + i % R);
        __syncthreads();
        for (uint32_t row = warp; row < R; row += W) {
            float m = -INFINITY, l = 0;
            for (uint32_t c = lane; c < count[k]; c += 32) m = fmaxf(m, ml[c * R + row].x);
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            for (uint32_t c = lane; c < count[k]; c += 32) {
                const float2 x = ml[c * R + row];
                const float w = x.x == m ? 1.0f : ex2(x.x - m);
                ml[c * R + row].x = w;
                l = fmaf(x.y, w, l);
            }
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
            if (lane == 0) sh.total[row] = l;
        }
        __syncthreads();
        for (uint32_t f = tid; f < NF * 32; f += W * 32) {
            const uint32_t row = row_of(f);
            float4 o = make_float4(0, 0, 0, 0);
            for (uint32_t c0 = 0; c0 < count[k]; c0 += 8) {
                float4 x[8];
#pragma unroll
                for (int c = 0; c < 8; c++) x[c] = __ldcg(reinterpret_cast<const float4*>(part_at(first_cta[k] + min(c0 + c, count[k] - 1), c0 + c == 0)) + f);
#pragma unroll
                for (int c = 0; c < 8; c++) {
                    if (c0 + c >= count[k]) break;
                    const float w = ml[(c0 + c) * R + row].x;
                    o.x = fmaf(x[c].x, w, o.x); o.y = fmaf(x[c].y, w, o.y); o.z = fmaf(x[c].z, w, o.z); o.w = fmaf(x[c].w, w, o.w);
                }
            }
            const float l = sh.total[row];
            store_out(open_job[k], f, o, l);
        }
        __syncthreads();
    }
}

size_t kv4_part_floats(uint32_t dim, int num_sms) { return (size_t)num_sms * 2 * (16 * dim + 32); }

namespace {
template <int NB, int R>
cudaError_t launch(const Kv4AttnArgs& a, int num_sms, cudaStream_t st, bool pdl) {
    using C = Cfg<NB, R>;
    static bool done[64] = {};
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return err;
    if (dev >= 64 || !done[dev]) {
        err = cudaFuncSetAttribute(kv4_attn_kernel<NB, R>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(typename C::Smem));
        if (err != cudaSuccess) return err;
        if (dev < 64) done[dev] = true;
    }
    cudaLaunchConfig_t lc = {}; cudaLaunchAttribute at[1];
    lc.gridDim = dim3(num_sms < (int)MAX_CTAS ? num_sms : (int)MAX_CTAS); lc.blockDim = dim3(C::WARPS * 32); lc.dynamicSmemBytes = sizeof(typename C::Smem); lc.stream = st;
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = at; lc.numAttrs = pdl ? 1 : 0;
    return cudaLaunchKernelEx(&lc, kv4_attn_kernel<NB, R>, a);
}
}  // namespace

cudaError_t launch_kv4_attention(const Kv4AttnArgs& a, uint32_t rows, uint32_t jobs, int num_sms, cudaStream_t st, bool pdl) {
    if (!jobs) return cudaSuccess;
    switch (a.shape.dim * 100 + rows) {
        case 6404: return launch<2, 4>(a, num_sms, st, pdl);
        case 6408: return launch<2, 8>(a, num_sms, st, pdl);
        case 6416: return launch<2, 16>(a, num_sms, st, pdl);
        case 12804: return launch<4, 4>(a, num_sms, st, pdl);
        case 12808: return launch<4, 8>(a, num_sms, st, pdl);
        case 12816: return launch<4, 16>(a, num_sms, st, pdl);
        case 25604: return launch<8, 4>(a, num_sms, st, pdl);
        case 25608: return launch<8, 8>(a, num_sms, st, pdl);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace alice
