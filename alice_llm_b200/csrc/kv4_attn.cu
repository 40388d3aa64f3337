// Attention of one or several new tokens over the 4-bit cache (csrc/kv4.cuh).
//
// A warp takes a job's 4, 8 or 16 (token, query head) rows against tiles of 16 keys with m16n8k16 products in half precision:
//   scores^T [key][row]  = sum over blocks of d * (codes . q), and m * (sum of q) of all blocks as a product of its own
//   out^T [dim][row]    += codes * (p * d), and m * p apart in f32
// with d, m a block's step and minimum. Codes of values enter less 8 (and m is m + 8 d), so that the two parts of a sum over many keys do
// not cancel; unpacking two of them is a mask and an exact addition in half precision. (Masked bits alone are exact operands too, as numbers
// below 2^-14, but the products of those lose bits in the sum: results were 4e-5 to 4e-4 off.) The other operand, q or p * d, is a pair of half-precision
// numbers (value and remainder, 22 bits), scaled by powers of two into the middle of their range: queries by one for a row, steps by one for each block of 32 dims.
// With up to 4 rows the pair fills two columns of the product, with more they are two products.
//
// All tiles of all jobs and key heads are one row of work that is cut into equal parts, a CTA an SM and again among its warps, so batches of any
// lengths are even. A warp streams its tiles through a ring of its own (cp.async); rows that several warps or CTAs had a part in are
// joined in shared memory, then by the CTA that is the last to bring its part.
//
// Weighted sums go to f32 sums every 8 tiles: products on tensor cores add up with less than f32 rounding, which over a long chain would add up itself. What is
// added up until then is of one magnitude: its weights have a reference of their own, the largest score of its first tiles, which moves when a score exceeds it by 2^8 or
// when the next sums begin with all of a row's 2^8 below it, and its steps lie within 2^8 (what is heavier, or larger, and comes elsewhere takes no bits from it). Where the
// steps of two tiles side by side lie further apart (a block of zeros with a weight counts too), these tiles' products are made in f32 by the ordinary pipes: 270 us where that is
// so in all of 131008 positions. One power of two for all blocks and for all that came before took 64 us instead of 69 there, and with values 2^20 apart was 1 to 5 % off.
//
// Bound by latency with few warps: two (R = 4: three) a quarter of an SM by registers, issue slots 47 % (57), tensor pipe 24 % (16), stalls led by fixed latencies of dependent
// instructions; start, merges and the join are 12 to 15 us of a large call. Measured, heads of 128: one token of 64 x 8 heads behind 131007 positions (168 MB) 69 us, one each
// of 64 users with 32 x 8 heads behind up to 4095 61 us.
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"
#include "kv4.cuh"
#include "kv4_query.cuh"

namespace alice {

namespace {

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

constexpr int STAGES = 4;
constexpr uint32_t FLUSH = 8;        // tiles (131008 positions: 4 tiles 1.2e-6 off and 76 us, 8 1.6e-6 and 69.6, 16 2.4e-6 and 67.8)
constexpr float ROOM = 8.0f;         // what a score may exceed the reference by, and what all scores of a row may be below it, in powers of two
constexpr float LIFT = 7.0f;         // weights are 2^7 times as large as they are (sums of them too): up to 2^15

// Parts of a row's sums brought to one reference, N at a time.
template <int N>
struct Joined {
    float m = -INFINITY, l = 0;
    float4 sum = make_float4(0, 0, 0, 0);
    __device__ __forceinline__ void add(const float2 (&ml)[N], const float4 (&x)[N], int n) {      // the first n count
        float top = m;
#pragma unroll
        for (int j = 0; j < N; j++) top = fmaxf(top, j < n ? ml[j].x : -INFINITY);
        float c = m == top ? 1.0f : ex2(m - top);
        l *= c; sum.x *= c; sum.y *= c; sum.z *= c; sum.w *= c;
        m = top;
#pragma unroll
        for (int j = 0; j < N; j++) {
            if (j >= n) continue;
            c = ml[j].x == top ? 1.0f : ex2(ml[j].x - top);
            l = fmaf(ml[j].y, c, l);
            sum.x = fmaf(x[j].x, c, sum.x); sum.y = fmaf(x[j].y, c, sum.y); sum.z = fmaf(x[j].z, c, sum.z); sum.w = fmaf(x[j].w, c, sum.w);
        }
    }
};

// A warp's part of a job that is not all of it.
struct Segment {
    uint32_t head;
    uint32_t job, row, first;
    uint16_t rows, ends;                 // 1: has the job's first tile, 2: its last; 4: there is one
};

template <int NB, int R>
struct Cfg {
    static constexpr bool SPLIT = R == 4;
    static constexpr int NT = R == 16 ? 2 : 1;                    // eight-column products
    static constexpr int RT = SPLIT ? 1 : 2 * NT;                 // rows a lane has scores and outputs of
    static constexpr int TP = R == 16 || NB == 8 ? 1 : 2;         // tiles taken together, as many as the registers hold (131008 positions: 65.6 us, one 68.2)
    // As many as the registers hold; of 4 rows 12 (56.7 us, 16 58.6 where a CTA has more to merge), of 8 as few as keep the products busy (12 no faster).
    static constexpr int WARPS = NB == 8 ? (R == 4 ? 8 : 6) : R == 4 ? 12 : 8;
    static constexpr uint32_t DIM = 32 * NB, TILE = kv4_tile_bytes(DIM);
    static constexpr int NF = NB * RT;                            // float4 of output a lane has
    static constexpr uint32_t PART = R * DIM + 2 * R;             // floats of a part of a job
    struct Smem {
        float4 sum[WARPS][2][NF][32];
        float2 ml[WARPS][2][R];                                   // reference and sum of weights
        Segment seg[2 * WARPS];
        float aside[WARPS * R * (NB + 1)];                        // of a job's queries: what is beside their operands
        uint32_t last[2];
        alignas(16) uint8_t ring[WARPS][STAGES][TILE];
    };
};

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the same with a sum that starts at zero
__device__ __forceinline__ void mma_f16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, const float (&z)[4]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(z[0]), "f"(z[1]), "f"(z[2]), "f"(z[3]));
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }    // -126 <= e <= 127
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

// half-precision number i of a lane's words
template <int N>
__device__ __forceinline__ float half_of(const Words<N>& x, int i) { return i & 1 ? __high2float(bits_half2(x.w[i / 2])) : __low2float(bits_half2(x.w[i / 2])); }

// The job that tile x of a key head belongs to: the last with job_tile <= x. All lanes look, 32 places at a time.
__device__ __forceinline__ uint32_t find_job(const uint32_t* job_tile, uint32_t jobs, uint32_t x, uint32_t lane) {
    uint32_t lo = 0, n = jobs;
    while (n > 1) {
        const uint32_t step = (n + 31) / 32, i = lo + lane * step;
        const uint32_t hit = __ballot_sync(0xffffffffu, lane * step < n && job_tile[i] <= x);
        const uint32_t k = 31 - __clz(hit);
        n = min(step, n - k * step);
        lo += k * step;
    }
    return lo;
}

}  // namespace

template <int NB, int R>
__global__ void __launch_bounds__(Cfg<NB, R>::WARPS * 32, 1) kv4_attn_kernel(const __grid_constant__ Kv4AttnArgs a) {
    using C = Cfg<NB, R>;
    constexpr int NT = C::NT, RT = C::RT, NF = C::NF, W = C::WARPS, TP = C::TP;
    constexpr bool SPLIT = C::SPLIT;
    constexpr uint32_t DIM = C::DIM, TILE = C::TILE;
    static_assert(sizeof(typename C::Smem) <= 227 * 1024 && NB >= 2, "");
    extern __shared__ __align__(16) uint8_t raw[];
    auto& sh = *reinterpret_cast<typename C::Smem*>(raw);
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    pdl_launch_dependents();
    pdl_wait();
    const Kv4Plan& pl = a.plan;
    const Kv4Head hd = *pl.head;
    if (!kv4_fits(hd, a)) return;
    const Kv4Job* const jobs = pl.job + hd.prompt_jobs;
    // Equal parts for the CTAs, those of one job only (a sequence of few new tokens) at the borders of key heads: no CTA has parts of two
    // of them then, and where a CTA can have all of a head there is nothing to join between CTAs.
    const uint32_t tiles = hd.tiles, total = tiles * a.shape.kv_heads, cta = blockIdx.x;
    uint32_t grid, splits = 0, c0, c1;
    if (hd.jobs == 1 && a.shape.kv_heads <= gridDim.x) {
        splits = tiles <= 2 * W ? 1 : min(gridDim.x / a.shape.kv_heads, (tiles + W - 1) / W);
        grid = splits * a.shape.kv_heads;
        const uint32_t h = cta / splits, i = cta - h * splits, per = tiles / splits, more = tiles - per * splits;
        c0 = h * tiles + i * per + min(i, more);
        c1 = c0 + per + (i < more ? 1 : 0);
    } else {
        grid = min(gridDim.x, (total + W - 1) / W);
        if (grid == 0) return;
        const uint32_t per = total / grid, more = total - per * grid;
        c0 = cta * per + min(cta, more);
        c1 = c0 + per + (cta < more ? 1 : 0);
    }
    if (cta >= grid) return;
    const uint32_t w0 = c0 + (c1 - c0) * warp / W, w1 = c0 + (c1 - c0) * (warp + 1) / W;
    if (lane < 2) sh.seg[2 * warp + lane].ends = 0;
    float zero[4];       // registers of their own: the start of a product's sums
#pragma unroll
    for (int i = 0; i < 4; i++) asm volatile("mov.f32 %0, 0f00000000;" : "=f"(zero[i]));

    if (w0 < w1) {
        // ---- the ring: tiles are asked for STAGES - 1 ahead ----
        const uint32_t ring = smem_u32(sh.ring[warp][0]);
        const uint32_t per_page = a.shape.tiles();
        uint32_t p_head = w0 / tiles, p_tile = w0 - p_head * tiles;
        uint32_t p_job = find_job(pl.job_tile, hd.jobs, p_tile, lane);
        uint32_t job = p_job, head = p_head;
        uint32_t p_seq = 0, p_tile0 = 0, p_end = 0, p_pages = 0, p_base = 0xffffffffu;    // of the job; pages of 32 pages, a lane each
        uint32_t p_left = 0;                                                             // tiles to come of the page and the job
        const uint8_t* p_src = nullptr;
        uint32_t p_count = w1 - w0;
        bool p_new = true;
        uint32_t p_n = 0, p_in = 0;
        auto look = [&]() {          // asks for the page of the next tile,
            if (p_new) {
                const Kv4Job nj = jobs[p_job];
                p_seq = nj.seq; p_tile0 = nj.tile0; p_end = nj.tile1;
                p_base = 0xffffffffu; p_new = false;
            }
            const uint32_t i = p_tile - p_tile0;
            p_n = i / per_page; p_in = i - p_n * per_page;
            if (p_base == 0xffffffffu || p_n >= p_base + 32) {
                p_base = p_n;
                p_pages = pl.table[(size_t)p_seq * pl.table_ld + min(p_n + lane, (p_end - 1 - p_tile0) / per_page)];
            }
        };
        auto found = [&]() {         // and has it
            const uint32_t page = __shfl_sync(0xffffffffu, p_pages, p_n - p_base);
            p_src = a.pool + (((size_t)page * a.shape.kv_heads + p_head) * per_page + p_in) * TILE + lane * 16;
            p_left = min(per_page - p_in, p_end - p_tile);
        };
        auto ask = [&](uint32_t stage) {
            if (p_count) {
                p_count--;
                if (p_left == 0) { look(); found(); }
                const uint32_t dst = ring + stage * TILE + lane * 16;
#pragma unroll
                for (uint32_t c = 0; c < (TILE / 16 + 31) / 32; c++)
                    if (TILE % 512 == 0 || c * 512 + lane * 16 < TILE) cp16(dst + c * 512, p_src + c * 512);
                p_src += TILE; p_tile++;
                if (--p_left == 0 && p_tile == p_end) {
                    p_new = true; p_job++;
                    if (p_tile == tiles) { p_tile = 0; p_job = 0; p_head++; }
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };

        look();
        uint32_t stage = 0, slot = 0;
        // The first tiles are asked for behind the first queries and their angles, which would wait for all of them otherwise; as few as the ring
        // holds behind the queries alone (24 short sequences of 64 dims 23.1 us, else 23.4; 131008 positions, where only the code differs, 63.6 and 66.2).
        const bool few = w1 - w0 <= STAGES;
        for (uint32_t at = w0; at < w1;) {
            // ---- a job, or this warp's part of it ----
            const Kv4Job jb = jobs[job];
            const uint32_t j0 = head * tiles + jb.tile0, j1 = head * tiles + jb.tile1, end = min(j1, w1);
            const bool has_first = at == j0, has_last = end == j1;

            // Queries: rotated, scaled, cut into pairs row by row, then read back as columns of the product in the order of a lane's codes. The
            // place is that of the job's sums, which have not begun.
            uint32_t qf[NT][NB][SPLIT ? 4 : 8];      // [..][0..3]: values (or by column values and remainders), [4..7]: remainders
            uint32_t qm[NT][2];                      // sums of a block's queries, likewise: against the minima
            float factor[RT];
            {
                constexpr uint32_t CH = R * DIM / 128, PER = DIM / 4 < 32 ? DIM / 4 : 32;      // pieces of 128 floats; lanes of a row
                const uint32_t place = smem_u32(&sh.sum[warp][slot][0][0]);      // [row][value, remainder][block][t][4 words]
                float* const aside = sh.aside + warp * R * (NB + 1);             // [row][sums of blocks, factor]
                float4 x[CH];
                uint32_t of[CH];          // row of the rotation table
#pragma unroll
                for (uint32_t c = 0; c < CH; c++) {
                    const uint32_t at_c = c * 128 + lane * 4, row = at_c / DIM, dim0 = at_c % DIM;
                    const uint32_t r = jb.row + min(row, jb.rows - 1), tok = r / a.group, at_tok = jb.first + tok;
                    x[c] = *reinterpret_cast<const float4*>(a.q + at_tok * a.q_ld + (size_t)(head * a.group + r - tok * a.group) * DIM + dim0);
                    of[c] = a.rope.by_token ? at_tok : jb.past + tok;
                }
                if (at == w0 && few) {
                    found();
#pragma unroll
                    for (int i = 0; i < STAGES; i++) ask(i);
                }
                if (a.rope.dims) {
                    constexpr uint32_t PER_ROW = DIM > 128 ? DIM / 128 : 1;
                    Turn w[PER_ROW];
#pragma unroll
                    for (uint32_t c = 0; c < CH; c += PER_ROW) {
#pragma unroll
                        for (uint32_t k = 0; k < PER_ROW; k++)      // rows of one token share it
                            if (c == 0 || of[c] != of[c >= PER_ROW ? c - PER_ROW : 0]) w[k] = turn_at(a.rope.table + (size_t)of[c] * a.rope.dims, lane * 4 % DIM + 128 * k, a.rope);
                        float4 y[PER_ROW];
#pragma unroll
                        for (uint32_t k = 0; k < PER_ROW; k++) y[k] = x[c + k];
#pragma unroll
                        for (uint32_t k = 0; k < PER_ROW; k++) x[c + k] = rotated4(y, k, lane * 4 % DIM + 128 * k, w[k], a.rope);
                    }
                }
                __syncwarp();
#pragma unroll
                for (uint32_t c = 0; c < CH; c++) {
                    const uint32_t at_c = c * 128 + lane * 4, row = at_c / DIM, b = at_c % DIM / 32;
                    const float f = row < jb.rows ? a.scale : 0.0f;
                    float v[4] = {x[c].x * f, x[c].y * f, x[c].z * f, x[c].w * f};
                    float top = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
                    if (DIM == 256) {      // the other half of the row
                        const float4 y = x[c ^ 1];
                        top = fmaxf(top, fmaxf(fmaxf(fabsf(y.x * f), fabsf(y.y * f)), fmaxf(fabsf(y.z * f), fabsf(y.w * f))));
                    }
#pragma unroll
                    for (uint32_t o = 1; o < PER; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                    int e2 = (int)((__float_as_uint(top) >> 23) & 0xff) - 127 - 9;     // the largest into 2^9 .. 2^10
                    e2 = min(max(e2, -100), 120);
                    const float down = pow2(-e2);
                    float sum = 0;
#pragma unroll
                    for (int e = 0; e < 4; e++) { v[e] *= down; sum += v[e]; }
#pragma unroll
                    for (int o = 1; o < 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                    if (lane % 8 == 0) aside[row * (NB + 1) + b] = sum;
                    if (at_c % DIM == 0) aside[row * (NB + 1) + NB] = pow2(e2) * 1.44269504088896341f;
                    // dims 8 t + e and 8 t + e + 4 share a word: with the neighbouring lane's
                    const __half2 h01 = __floats2half2_rn(v[0], v[1]), h23 = __floats2half2_rn(v[2], v[3]);
                    const float2 f01 = __half22float2(h01), f23 = __half22float2(h23);
                    const uint32_t mine[2][2] = {{half2_bits(h01), half2_bits(h23)},
                                                 {half2_bits(__floats2half2_rn(v[0] - f01.x, v[1] - f01.y)), half2_bits(__floats2half2_rn(v[2] - f23.x, v[3] - f23.y))}};
                    const bool odd = lane & 1;
#pragma unroll
                    for (int part = 0; part < 2; part++) {
                        const uint32_t got = __shfl_xor_sync(0xffffffffu, mine[part][odd ? 0 : 1], 1), keep = mine[part][odd ? 1 : 0];
                        // even lane: words 0, 1 of (its, the other's); odd: words 2, 3 of (the other's, its)
                        const uint32_t lo = odd ? got : keep, hi = odd ? keep : got;
                        const uint32_t to = place + ((row * 2 + part) * NB + b) * 64 + (lane % 8 / 2) * 16 + (odd ? 8 : 0);
                        asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(to), "r"(__byte_perm(lo, hi, 0x5410)), "r"(__byte_perm(lo, hi, 0x7632)) : "memory");
                    }
                }
                __syncwarp();
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    const uint32_t row = SPLIT ? g >> 1 : n * 8 + g;
#pragma unroll
                    for (int b = 0; b < NB; b++)
#pragma unroll
                        for (int part = 0; part < (SPLIT ? 1 : 2); part++) {
                            const uint4 w = lds128(place + ((row * 2 + (SPLIT ? g & 1 : part)) * NB + b) * 64 + t * 16);
                            qf[n][b][part * 4] = w.x; qf[n][b][part * 4 + 1] = w.y; qf[n][b][part * 4 + 2] = w.z; qf[n][b][part * 4 + 3] = w.w;
                        }
                    // The minima of a key are the first columns (of 8 blocks all) of an operand's 16, again as the next; the sums' values and
                    // remainders stand against them.
                    const uint32_t p = NB == 8 ? t : t % (NB / 2);
                    const float s0 = aside[row * (NB + 1) + 2 * p], s1 = aside[row * (NB + 1) + 2 * p + 1];
                    const __half2 hi = __floats2half2_rn(s0, s1);
                    const float2 back = __half22float2(hi);
                    const uint32_t value = half2_bits(hi), left = half2_bits(__floats2half2_rn(s0 - back.x, s1 - back.y));
                    qm[n][0] = NB == 8 || t < NB / 2 ? value : t < NB ? left : 0;
                    qm[n][1] = NB == 8 ? left : 0;
                    if (SPLIT && (g & 1)) qm[n][0] = qm[n][1] = 0;
                }
#pragma unroll
                for (int i = 0; i < RT; i++) factor[i] = aside[(SPLIT ? t : (i >> 1) * 8 + 2 * t + (i & 1)) * (NB + 1) + NB];
                __syncwarp();
            }
            if (at == w0 && !few) {
                found();
#pragma unroll
                for (int i = 0; i < STAGES; i++) ask(i);
            }
            const uint32_t to_key = (end - j0) * KV4_TILE;      // of this warp's part
            uint32_t limit[RT], least = to_key, far = 0;        // positions a row sees, of this part
#pragma unroll
            for (int i = 0; i < RT; i++) {
                const uint32_t row = SPLIT ? t : (i >> 1) * 8 + 2 * t + (i & 1);
                limit[i] = row < jb.rows ? min(to_key, jb.past + (jb.row + row) / a.group + 1) : 0u;
                if (row < jb.rows) least = min(least, limit[i]);
                far = max(far, limit[i]);
            }
            least = __reduce_min_sync(0xffffffffu, least);
            far = __reduce_max_sync(0xffffffffu, far);

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
            // Steps in acc, by block of dims (two to a register): as half-precision bits less `least_d` they have none of the bits `too_far`; 2^(14 - e) that they are
            // multiplied by, e in bytes of last_e.
            // A borrow of the lower half is one that is too far itself, or from NO_STEP, and then the upper half is taken one higher than it is: no harm at its ends.
            constexpr uint32_t NO_STEP = 0xe001e001u, NOTHING = 0x7fff7fffu, FAR = 0xe000e000u;      // 0 and nothing else; no step at all
            uint32_t least_d[NB / 2], too_far[NB / 2], last_e[NB / 4 ? NB / 4 : 1];
            __half2 dscale[NB / 2];
            auto no_steps = [&]() {
#pragma unroll
                for (int b = 0; b < NB / 2; b++) { least_d[b] = NOTHING; too_far[b] = FAR; dscale[b] = __float2half2_rn(0.0f); }
            };
            no_steps();
#pragma unroll
            for (int b = 0; b < NB; b += 4) last_e[b / 4] = 0;
            uint32_t held = 0;                  // tiles in acc
            bool begun = false;                 // sums are in shared memory
            float4* const mine = &sh.sum[warp][slot][0][lane];

            // what acc, accm and l hold joins the sums in shared memory
            auto flush = [&]() {
#pragma unroll
                for (int i = 0; i < RT; i++) {
                    const float top = fmaxf(mref[i], ref[i]), c = mref[i] == top ? 1.0f : ex2(mref[i] - top), f = ref[i] == top ? 1.0f : ex2(ref[i] - top);
                    float s = l[i];
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
                    lsum[i] = fmaf(lsum[i], c, s * f);
                    l[i] = 0; mref[i] = top;
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        const float back = pow2((int)(last_e[b / 4] >> 8 * (b % 4) & 31) - 14) * f;
                        float am = accm[i][b];
#pragma unroll
                        for (int o = 4; o < 32; o <<= 1) am += __shfl_xor_sync(0xffffffffu, am, o);
                        am *= f;
                        accm[i][b] = 0;
                        float v[4];
#pragma unroll
                        for (int u = 0; u < 2; u++) {
                            float (&x)[4] = acc[SPLIT ? 0 : i >> 1][b][u];
                            if (SPLIT) { v[2 * u] = x[0] + x[1]; v[2 * u + 1] = x[2] + x[3]; x[0] = x[1] = x[2] = x[3] = 0; }
                            else { v[2 * u] = x[i & 1]; v[2 * u + 1] = x[2 + (i & 1)]; x[i & 1] = x[2 + (i & 1)] = 0; }
                        }
                        float4 o = make_float4(fmaf(v[0], back, am), fmaf(v[1], back, am), fmaf(v[2], back, am), fmaf(v[3], back, am));
                        float4* to = mine + (i * NB + b) * 32;
                        if (begun) { const float4 p = *to; o.x = fmaf(p.x, c, o.x); o.y = fmaf(p.y, c, o.y); o.z = fmaf(p.z, c, o.z); o.w = fmaf(p.w, c, o.w); }
                        *to = o;
                    }
                }
                held = 0; begun = true;
            };

            uint32_t key0 = (at - j0) * KV4_TILE;
            while (at < end) {
                asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - TP) : "memory");
                __syncwarp();
                uint32_t base[TP];
#pragma unroll
                for (int x = 0; x < TP; x++) base[x] = ring + (stage + x) % STAGES * TILE;
                float s[TP][RT][2];             // of keys tau(g), 8 + tau(g)
                // ---- scores: the minima's part, then block by block ----
#pragma unroll
                for (int x = 0; x < TP; x++) {
                    const uint32_t mat = base[x] + kv4_k_scales(DIM) + g * (4 * NB) + 2 * NB + 4 * (t % (NB / 2)), ma = lds32(mat), mb = lds32(mat + 32 * NB);
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        float c[4];
                        mma_f16_first(c, ma, mb, ma, mb, qm[n][0], qm[n][1], zero);
                        if (SPLIT) { s[x][0][0] = c[0]; s[x][0][1] = c[2]; }
                        else {
#pragma unroll
                            for (int j = 0; j < 2; j++) { s[x][(2 * n + j) % RT][0] = c[j]; s[x][(2 * n + j) % RT][1] = c[2 + j]; }
                        }
                    }
                }
#pragma unroll
                for (int h = 0; h < (NB + 3) / 4; h++) {
                    constexpr int NW = NB < 4 ? NB : 4;
                    Words<NW> ka[TP], kb[TP];
                    Words<NW / 2> sa[TP], sb[TP];
#pragma unroll
                    for (int x = 0; x < TP; x++) {
                        const uint32_t kat = base[x] + g * (DIM / 2) + (NB == 8 ? h * 64 + t * 16 : t * NB * 4), srow = base[x] + kv4_k_scales(DIM) + g * (4 * NB) + h * 8;
                        ka[x] = lds_words<NW>(kat); kb[x] = lds_words<NW>(kat + 4 * DIM);
                        sa[x] = lds_words<NW / 2>(srow); sb[x] = lds_words<NW / 2>(srow + 32 * NB);
                    }
                    // two blocks of every tile side by side: a product's sum is waited for by the next one of its chain
#pragma unroll
                    for (int w = 0; w < NW; w += 2) {
                        Codes xa[2][TP], xb[2][TP];
                        float c[2][TP][NT][4];
#pragma unroll
                        for (int u = 0; u < 2; u++)
#pragma unroll
                            for (int x = 0; x < TP; x++) { xa[u][x] = unpack<0>(ka[x].w[w + u]); xb[u][x] = unpack<0>(kb[x].w[w + u]); }
#pragma unroll
                        for (int step = 0; step < (SPLIT ? 2 : 4); step++)
#pragma unroll
                            for (int u = 0; u < 2; u++)
#pragma unroll
                                for (int x = 0; x < TP; x++)
#pragma unroll
                                    for (int n = 0; n < NT; n++) {
                                        const int b = h * 4 + w + u, o = step & 1 ? 2 : 0;
                                        const uint32_t q0 = qf[n][b][SPLIT ? o : 2 * step], q1 = qf[n][b][SPLIT ? o + 1 : 2 * step + 1];
                                        if (step == 0) mma_f16_first(c[u][x][n], xa[u][x].v[o], xb[u][x].v[o], xa[u][x].v[o + 1], xb[u][x].v[o + 1], q0, q1, zero);
                                        else mma_f16(c[u][x][n], xa[u][x].v[o], xb[u][x].v[o], xa[u][x].v[o + 1], xb[u][x].v[o + 1], q0, q1);
                                    }
#pragma unroll
                        for (int u = 0; u < 2; u++)
#pragma unroll
                            for (int x = 0; x < TP; x++) {
                                const float da = half_of(sa[x], w + u), db = half_of(sb[x], w + u);
#pragma unroll
                                for (int n = 0; n < NT; n++) {
                                    const float (&y)[4] = c[u][x][n];
                                    if (SPLIT) {
                                        s[x][0][0] = fmaf(da, y[0] + y[1], s[x][0][0]);
                                        s[x][0][1] = fmaf(db, y[2] + y[3], s[x][0][1]);
                                    } else {
#pragma unroll
                                        for (int j = 0; j < 2; j++) {
                                            const int i = (2 * n + j) % RT;
                                            s[x][i][0] = fmaf(da, y[j], s[x][i][0]);
                                            s[x][i][1] = fmaf(db, y[2 + j], s[x][i][1]);
                                        }
                                    }
                                }
                            }
                    }
                }
                // ---- weights ----
                const uint32_t tau = (g >> 1) + 4 * (g & 1), key = key0 + tau;
                Words<NB> va[TP], vb[TP];       // scales of the values
#pragma unroll
                for (int x = 0; x < TP; x++) {
                    const uint32_t vsrow = base[x] + kv4_v_scales(DIM) + g * (4 * NB);
                    va[x] = lds_words<NB>(vsrow); vb[x] = lds_words<NB>(vsrow + 32 * NB);
                }
                bool begin_anew = false;         // what is held goes to shared memory first, and these tiles are looked at again
                auto weights = [&](auto edge_t) {
                    constexpr bool edge = decltype(edge_t)::value;       // some row does not see all of the tiles
                    bool move = false;
                    uint32_t beyond[NB / 2] = {}, too = 0;
#pragma unroll
                    for (int i = 0; i < RT; i++) {
                        float m = -INFINITY;
#pragma unroll
                        for (int x = 0; x < TP; x++)
#pragma unroll
                            for (int k = 0; k < 2; k++) {
                                if (edge && key + 16 * x + 8 * k >= limit[i]) s[x][i][k] = -INFINITY;
                                m = fmaxf(m, s[x][i][k]);
                            }
                        move |= m * factor[i] > ref[i] + ROOM;
                        if (held == 0) move |= !(__ballot_sync(0xffffffffu, m * factor[i] > ref[i] - ROOM) & 0x11111111u << t);      // none of the row's
                    }
#pragma unroll
                    for (int x = 0; x < TP; x++)
#pragma unroll
                        for (int k = 0; k < 2; k++)
#pragma unroll
                            for (int b = 0; b < NB / 2; b++) {
                                uint32_t& d = (k ? vb : va)[x].w[b];
                                const bool none = edge && key + 16 * x + 8 * k >= far;      // keys that no row sees: whatever lies there has no part
                                if (none) d = 0;
                                beyond[b] |= none ? 0 : d - least_d[b];
                            }
                    uint32_t hi[NB / 2], lo[NB / 2];
                    auto outside = [&]() {
                        bool out = false;
#pragma unroll
                        for (int b = 0; b < NB / 2; b++) out |= __vcmpgtu2(hi[b], __vadd2(least_d[b], ~too_far[b])) || __vcmplts2(lo[b], least_d[b]);
                        return out;
                    };
#pragma unroll
                    for (int b = 0; b < NB / 2; b++) too |= beyond[b] & too_far[b];
                    bool again = __any_sync(0xffffffffu, move || too);
                    if (again) {
                        // The largest steps and the least; a step of 0 has the size of its minimum, and a NaN's is above all.
#pragma unroll
                        for (int b = 0; b < NB / 2; b++) {
                            hi[b] = 0; lo[b] = 0x7fff7fffu;
#pragma unroll
                            for (int x = 0; x < TP; x++)
#pragma unroll
                                for (int k = 0; k < 2; k++) {
                                    if (edge && key + 16 * x + 8 * k >= far) continue;
                                    const uint32_t d = (k ? vb : va)[x].w[b], m = (k ? vb : va)[x].w[NB / 2 + b] & 0x7fff7fffu;
                                    hi[b] = __vmaxu2(hi[b], d); lo[b] = __vminu2(lo[b], d | m & __vcmpeq2(d, 0));
                                }
                        }
                        again = __any_sync(0xffffffffu, move || outside());
                    }
                    if (again) {
                        if (held) { begin_anew = true; return; }
                        // A block by each of NB lanes. To below 1, with weights up to 2^15 then in range: by 2^(14 - e), e the exponent field that is the last within. That of the
                        // largest step is the one before, and the least is 2^-8 then. Of the steps below 2^-8 (fields 0 to 6) the least is 2^-4 to 2^-6 of the largest, and
                        // 2^-11 then.
                        uint32_t d = 0;
#pragma unroll
                        for (int b = 0; b < NB / 2; b++) {
                            uint32_t top = hi[b];
#pragma unroll
                            for (int o = 4; o < 32; o <<= 1) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, o));
                            if (lane / 2 % (NB / 2) == b) d = lane & 1 ? top >> 16 : top & 0xffff;
                        }
                        const uint32_t field = d >> 10;
                        uint32_t e = field + 1, least = (field - 6) << 10, far_bits = 0xe000;
                        if (field < 7) {
                            e = field >= 4 ? 8 : field >= 2 ? 4 : field + 1;
                            least = field >= 4 ? 512 : field >= 2 ? 64 : field ? 16 : max(d >> 6, 1u);
                            far_bits = field >= 4 ? 0xe000 : field >= 2 ? 0xf000 : field ? 0xf800 : 0xfc00;
                            if (!d) { least = NO_STEP & 0xffff; far_bits = 0xe000; }
                        }
                        const uint32_t range = least | far_bits << 16, power = (e <= 28 ? (29 - e) << 10 : 0x400u >> (e - 28)) | e << 16;
#pragma unroll
                        for (int b = 0; b < NB / 2; b++) {
                            const uint32_t r0 = __shfl_sync(0xffffffffu, range, 2 * b), r1 = __shfl_sync(0xffffffffu, range, 2 * b + 1), p0 = __shfl_sync(0xffffffffu, power, 2 * b),
                                           p1 = __shfl_sync(0xffffffffu, power, 2 * b + 1);
                            least_d[b] = __byte_perm(r0, r1, 0x5410); too_far[b] = __byte_perm(r0, r1, 0x7632); dscale[b] = bits_half2(__byte_perm(p0, p1, 0x5410));
                            const uint32_t es = (p0 >> 16 | p1 >> 16 << 8) << 16 * (b % 2);
                            last_e[b / 2] = b % 2 ? last_e[b / 2] | es : es;
                        }
#pragma unroll
                        for (int i = 0; i < RT; i++) {
                            float m = fmaxf(s[0][i][0], s[0][i][1]);
#pragma unroll
                            for (int x = 1; x < TP; x++) m = fmaxf(m, fmaxf(s[x][i][0], s[x][i][1]));
#pragma unroll
                            for (int o = 4; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                            if (m > -INFINITY) ref[i] = m * factor[i];
                        }
                        if (__any_sync(0xffffffffu, outside())) {
                            // Steps too far apart for one power of two: in f32 and without products, by the lanes that have the sums of these rows and dims.
#pragma unroll 1
                            for (uint32_t xk = 0; xk < 2 * TP; xk++) {
                                const uint32_t x = xk >> 1, k = xk & 1, tile = ring + (stage + x) % STAGES * TILE;
                                float p[RT];
#pragma unroll
                                for (int i = 0; i < RT; i++) {
                                    float v = k ? s[0][i][1] : s[0][i][0];
                                    if (TP == 2 && x) v = k ? s[TP - 1][i][1] : s[TP - 1][i][0];
                                    p[i] = edge && key + 8 * xk >= limit[i] ? 0.0f : ex2(fmaf(v, factor[i], LIFT - ref[i]));
                                }
#pragma unroll 1
                                for (uint32_t j = 0; j < 8 && key0 + 8 * xk + j < far; j++) {
                                    const uint32_t row = kv4_row(j);
                                    const Words<(NB + 1) / 2> codes = lds_words<(NB + 1) / 2>(tile + kv4_v_codes(DIM) + (8 * k + j) * (DIM / 2) + g * (2 * NB));
                                    const Words<NB / 2> d = lds_words<NB / 2>(tile + kv4_v_scales(DIM) + (8 * k + row) * (4 * NB));
#pragma unroll
                                    for (int i = 0; i < RT; i++) {
                                        const float w = __shfl_sync(0xffffffffu, p[i], 4 * row + t);
#pragma unroll
                                        for (int b = 0; b < NB; b++) {
                                            const float wd = w * half_of(d, b);
#pragma unroll
                                            for (int c = 0; c < 4; c++) {
                                                float& sum = acc[SPLIT ? 0 : i >> 1][b][c >> 1][c % 2 * 2 + (SPLIT ? 0 : i & 1)];
                                                sum = fmaf(wd, (float)(codes.w[b / 2] >> (16 * (b & 1) + 4 * c) & 15) - 8.0f, sum);
                                            }
                                        }
                                    }
                                }
                            }
#pragma unroll
                            for (int b = 0; b < NB; b += 4) last_e[b / 4] = 0x0e0e0e0eu;      // as they are
                            no_steps();              // no part in the products
                            held = FLUSH;            // and what comes next is by itself
                        }
                    }
#pragma unroll
                    for (int i = 0; i < RT; i++)
#pragma unroll
                        for (int x = 0; x < TP; x++) {
#pragma unroll
                            for (int k = 0; k < 2; k++) {
                                s[x][i][k] = ex2(fmaf(s[x][i][k], factor[i], LIFT - ref[i]));
                                if (edge && key + 16 * x + 8 * k >= limit[i]) s[x][i][k] = 0;
                            }
                            l[i] += s[x][i][0] + s[x][i][1];
                        }
                    // minima: of a key that a row does not see not even a NaN
#pragma unroll
                    for (int x = 0; x < TP; x++)
#pragma unroll
                        for (int b = 0; b < NB; b++) {
                            const float ma = fmaf(8.0f, half_of(va[x], b), half_of(va[x], NB + b)), mb = fmaf(8.0f, half_of(vb[x], b), half_of(vb[x], NB + b));   // what a code of 8 stands for
#pragma unroll
                            for (int i = 0; i < RT; i++) {
                                if (!edge) accm[i][b] = fmaf(s[x][i][0], ma, fmaf(s[x][i][1], mb, accm[i][b]));
                                else {
                                    if (key + 16 * x < limit[i]) accm[i][b] = fmaf(s[x][i][0], ma, accm[i][b]);
                                    if (key + 16 * x + 8 < limit[i]) accm[i][b] = fmaf(s[x][i][1], mb, accm[i][b]);
                                }
                            }
                        }
                };
                if (key0 + KV4_TILE * TP > least) weights(std::true_type{}); else weights(std::false_type{});
                if (!begin_anew) {
                    // ---- values: weight times step as a pair of half-precision numbers, from the weight's pair ----
#pragma unroll
                    for (int x = 0; x < TP; x++) {
                        Words<(NB + 1) / 2> v[4];
                        const uint32_t vrow = base[x] + kv4_v_codes(DIM) + t * (DIM / 2) + g * (2 * NB);
#pragma unroll
                        for (int i = 0; i < 4; i++) v[i] = lds_words<(NB + 1) / 2>(vrow + i * 2 * DIM);
                        __half2 ph[NT][2], pl[NT][2];       // of two rows, or of one twice
#pragma unroll
                        for (int n = 0; n < NT; n++)
#pragma unroll
                            for (int k = 0; k < 2; k++) {
                                const float p0 = s[x][SPLIT ? 0 : 2 * n % RT][k], p1 = s[x][SPLIT ? 0 : (2 * n + 1) % RT][k];
                                ph[n][k] = __floats2half2_rn(p0, p1);
                                const float2 back = __half22float2(ph[n][k]);
                                pl[n][k] = __floats2half2_rn(p0 - back.x, p1 - back.y);
                            }
#pragma unroll
                        for (int b2 = 0; b2 < NB / 2; b2++) {
                            const __half2 d2[2] = {__hmul2(bits_half2(va[x].w[b2]), dscale[b2]), __hmul2(bits_half2(vb[x].w[b2]), dscale[b2])};
                            Codes ca[2], cb[2];
#pragma unroll
                            for (int u = 0; u < 2; u++) {
                                const uint32_t pick = u ? 0x7632u : 0x5410u;
                                ca[u] = unpack<8>(__byte_perm(v[0].w[b2], v[1].w[b2], pick));
                                cb[u] = unpack<8>(__byte_perm(v[2].w[b2], v[3].w[b2], pick));
                            }
                            // w1 = p d to half precision, w2 = what is missing: p's value times d less w1 is exact
                            auto product = [](__half2 hi, __half2 lo, __half2 d, __half2& w1, __half2& w2) {
                                w1 = __hmul2(hi, d);
                                w2 = __hfma2(lo, d, __hfma2(hi, d, __hneg2(w1)));
                            };
                            if (SPLIT) {
                                __half2 w1[2], w2[2];
#pragma unroll
                                for (int k = 0; k < 2; k++) product(ph[0][k], pl[0][k], d2[k], w1[k], w2[k]);
#pragma unroll
                                for (int u = 0; u < 2; u++) {
                                    const uint32_t pick = u ? 0x7632u : 0x5410u;
                                    const uint32_t b0 = transposed(__byte_perm(half2_bits(w1[0]), half2_bits(w2[0]), pick)), b1 = transposed(__byte_perm(half2_bits(w1[1]), half2_bits(w2[1]), pick));
                                    mma_f16(acc[0][2 * b2 + u][0], ca[u].v[0], ca[u].v[1], cb[u].v[0], cb[u].v[1], b0, b1);
                                    mma_f16(acc[0][2 * b2 + u][1], ca[u].v[2], ca[u].v[3], cb[u].v[2], cb[u].v[3], b0, b1);
                                }
                            } else {
#pragma unroll
                                for (int u = 0; u < 2; u++)
#pragma unroll
                                    for (int n = 0; n < NT; n++) {
                                        __half2 w1[2], w2[2];
#pragma unroll
                                        for (int k = 0; k < 2; k++) product(ph[n][k], pl[n][k], u ? __high2half2(d2[k]) : __low2half2(d2[k]), w1[k], w2[k]);
                                        float (&o)[2][4] = acc[n][2 * b2 + u];
                                        const uint32_t b0 = transposed(half2_bits(w1[0])), b1 = transposed(half2_bits(w1[1])), e0 = transposed(half2_bits(w2[0])), e1 = transposed(half2_bits(w2[1]));
                                        mma_f16(o[0], ca[u].v[0], ca[u].v[1], cb[u].v[0], cb[u].v[1], b0, b1);
                                        mma_f16(o[1], ca[u].v[2], ca[u].v[3], cb[u].v[2], cb[u].v[3], b0, b1);
                                        mma_f16(o[0], ca[u].v[0], ca[u].v[1], cb[u].v[0], cb[u].v[1], e0, e1);
                                        mma_f16(o[1], ca[u].v[2], ca[u].v[3], cb[u].v[2], cb[u].v[3], e0, e1);
                                    }
                            }
                        }
                    }
                    __syncwarp();
                    ask(stage);
                    stage = (stage + 1) % STAGES; at++; held++; key0 += KV4_TILE;
                    if (TP == 2 && at < end) {
                        ask(stage);
                        stage = (stage + 1) % STAGES; at++; held++; key0 += KV4_TILE;
                    }
                }
                if (begin_anew || held >= FLUSH || at >= end) flush();
            }

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
                if (lane == 0) sh.seg[2 * warp + slot] = Segment{head, job, jb.row, jb.first, (uint16_t)jb.rows, (uint16_t)(4u | (has_first ? 1u : 0u) | (has_last ? 2u : 0u))};
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
    // Parts in the order of the work, a lane each; those of one job are a run.
    Segment sg{};
    if (lane < 2 * W) sg = sh.seg[lane];
    const uint32_t valid = __ballot_sync(0xffffffffu, sg.ends != 0), below = valid & ((1u << lane) - 1);
    if (!valid) return;
    const int before = below ? 31 - __clz(below) : 0;
    const uint32_t pj = __shfl_sync(0xffffffffu, sg.job, before), ph = __shfl_sync(0xffffffffu, sg.head, before);
    const uint32_t starts = __ballot_sync(0xffffffffu, sg.ends && (!below || pj != sg.job || ph != sg.head));
    const int runs = __popc(starts), run = __popc(starts & (0xffffffffu >> (31 - lane))) - 1;
    // a row's place in the fragments: element f = (i * NB + b) * 32 + lane
    auto row_of = [](uint32_t f) { const uint32_t i = f / (NB * 32), ln = f & 31; return SPLIT ? ln & 3 : (i >> 1) * 8 + 2 * (ln & 3) + (i & 1); };
    auto store_out = [&](const Segment& of, uint32_t f, float4 o, float l) {
        const uint32_t row = row_of(f);
        if (row >= of.rows) return;
        const uint32_t r = of.row + row, b = f / 32 % NB, tok = r / a.group;
        const float inv = 1.0f / l;
        float* out = a.out + (size_t)(of.first + tok) * a.out_ld + (size_t)(of.head * a.group + r - tok * a.group) * DIM + b * 32 + 4 * ((f & 31) >> 2);
        *reinterpret_cast<float4*>(out) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    };
    auto part_at = [&](uint32_t of, uint32_t which) { return a.part + ((size_t)of * 2 + which) * C::PART; };
    constexpr uint32_t NE = NF * 32;
    for (uint32_t i = tid; i < runs * NE; i += W * 32) {
        const uint32_t k = i / NE, f = i % NE, row = row_of(f);
        uint32_t members = __ballot_sync(0xffffffffu, sg.ends && run == (int)k);
        const uint32_t ends = __reduce_or_sync(0xffffffffu, run == (int)k ? (uint32_t)sg.ends : 0u), e0 = __ffs(members) - 1;
        Joined<4> o;
        while (members) {
            float2 ml[4];
            float4 x[4];
            int n = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t e = members ? __ffs(members) - 1 : e0;
                n += members != 0;
                ml[j] = sh.ml[e >> 1][e & 1][row];
                x[j] = (&sh.sum[e >> 1][e & 1][0][0])[f];
                members &= members - 1;
            }
            o.add(ml, x, n);
        }
        if ((ends & 3) == 3) store_out(sh.seg[e0], f, o.sum, o.l);
        else {
            float* to = part_at(cta, ends & 1);
            __stcg(reinterpret_cast<float4*>(to) + f, o.sum);
            if ((f / 32) % NB == 0 && (f & 31) < 4) __stcg(reinterpret_cast<float2*>(to + R * DIM) + row, make_float2(o.m, o.l));
        }
    }
    // Jobs that other CTAs have parts of: [0] one that began before this CTA, [1] one that begins in it. A lane of each warp finds the
    // same two.
    uint32_t open[2] = {0xffffffffu, 0xffffffffu};
    for (int k = 0; k < runs; k++) {
        const uint32_t ends = __reduce_or_sync(0xffffffffu, run == k ? sg.ends & 3u : 0u), e = __ffs(__ballot_sync(0xffffffffu, sg.ends && run == k)) - 1;
        if (ends == 1) open[1] = e;
        if (!(ends & 1)) open[0] = e;
    }
    if ((open[0] & open[1]) == 0xffffffffu) return;
    __threadfence();
    __syncthreads();
    uint32_t first_cta[2], count[2];
#pragma unroll
    for (int k = 0; k < 2; k++) {
        first_cta[k] = count[k] = 0;
        if (open[k] == 0xffffffffu) continue;
        const Segment& of = sh.seg[open[k]];
        if (splits) { first_cta[k] = of.head * splits; count[k] = splits; }
        else {
            const uint32_t per = total / grid, more = total - per * grid, wide = more * (per + 1);
            auto cta_of = [&](uint32_t x) { return x < wide ? x / (per + 1) : more + (x - wide) / per; };
            first_cta[k] = cta_of(of.head * tiles + jobs[of.job].tile0);
            count[k] = cta_of(of.head * tiles + jobs[of.job].tile1 - 1) - first_cta[k] + 1;
        }
        if (tid == 0 && atomicAdd(a.tickets + first_cta[k], 1u) == count[k] - 1) {
            a.tickets[first_cta[k]] = 0;
            sh.last[k] = 1;
        }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2; k++) {
        if (!sh.last[k]) continue;
        __threadfence();
        for (uint32_t f = tid; f < NE; f += W * 32) {
            constexpr int AT_ONCE = 10;
            const uint32_t row = row_of(f);
            Joined<AT_ONCE> o;
            for (uint32_t i = 0; i < count[k]; i += AT_ONCE) {
                float2 ml[AT_ONCE];
                float4 x[AT_ONCE];
#pragma unroll
                for (int j = 0; j < AT_ONCE; j++) {
                    const uint32_t c = min(i + j, count[k] - 1);
                    const float* from = part_at(first_cta[k] + c, c == 0);
                    ml[j] = __ldcg(reinterpret_cast<const float2*>(from + R * DIM) + row);
                    x[j] = __ldcg(reinterpret_cast<const float4*>(from) + f);
                }
                o.add(ml, x, (int)min(count[k] - i, (uint32_t)AT_ONCE));
            }
            store_out(sh.seg[open[k]], f, o.sum, o.l);
        }
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
    lc.gridDim = dim3(num_sms); lc.blockDim = dim3(C::WARPS * 32); lc.dynamicSmemBytes = sizeof(typename C::Smem); lc.stream = st;
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = at; lc.numAttrs = pdl ? 1 : 0;
    return cudaLaunchKernelEx(&lc, kv4_attn_kernel<NB, R>, a);
}
}  // namespace

cudaError_t launch_kv4_attention(const Kv4AttnArgs& a, int num_sms, cudaStream_t st, bool pdl) {
    if (a.prompt_jobs) {
        const cudaError_t err = launch_kv4_prompt(a, st, pdl);
        if (err != cudaSuccess || !a.rows) return err;
    }
    switch (a.shape.dim * 100 + a.rows) {
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
