// Attention of many new tokens over the 4-bit cache (csrc/kv4.cuh): 128 (token, query head) rows of a key head against 64 keys at a time, both
// products on the fifth-generation tensor cores.
//
// With a block's step d and minimum m a number is d * (code - 8) + (m + 8 d). Every factor is a pair of half-precision numbers (value and
// remainder, 22 bits; d * (code - 8) has 15) and a product three of them: value value, value remainder, remainder value. The second part is the same for
// the 32 dims of a block, so it is a few more columns of the operand, against the sums of a block's queries in one product and with sums of its
// own in the other. Of 256 keys both are scaled by a power of two to below 2^15: what is 2^18 and more below the largest of them has fewer than 22 bits, 2^-40 of that largest.
// Weights are 2^7 to 2^15 at a row's largest: those 2^-10 and less of it have fewer than 22 bits, 2^-31 of it. (Values 2^20 times as large as the others with weights of 1e-10: 4e-6 off,
// 2^30 times 4e-3; a key without a value that has all but 1e-7 of the weight: 4e-4. csrc/kv4_attn.cu has no such limits.)
//
// Twenty warps: one brings tiles of the pool (bulk copies, a ring of four blocks), one looks their scales over ahead of that (largest magnitude, NaN), four and four
// turn codes of keys and of values into operands in shared memory (2 instructions a number in half precision), two issue the products of the one and the other kind,
// so that one's waits are filled with the other's, and eight turn scores into weights, a row by a lane of two warps: half of a block's keys and half of the
// dims' sums each. Queries and weights lie in tensor memory, the weights where the scores were; scores of the next blocks run while weights are made. Sums of four
// blocks add up in tensor memory and go to registers then, in f32: over a long chain the tensor cores' sums would be further off than f32's. The
// reference of the weights moves as in csrc/kv4_attn.cu; what has been summed up in tensor memory moves with it.
//
// Measured: 2048 tokens x 32 heads of 128 (8 of keys) behind 1021 positions 210 us (the products alone: 124 at the measured bf16 rate; jobs of 16 rows on
// mma.sync: 715). A block takes 2600 clocks, the products 1630 of them: what is lost are the hand-overs from warps to warps. With operand warps that load from the pool
// themselves it was 667 us, with one warp a row, one for all products and every block's sums to registers 252, with warps that make both operands 6 us more.
//
// A cluster's CTAs share the keys of a job where there are fewer jobs than SMs, and join through distributed shared memory. A key or value
// that is NaN enters as zero, and rows that see it are NaN: those whose keys reach past the first such position.
//
// Every wait is bounded; tensor memory is given back, and products and copies are waited for, on all ways out.
#include "common.cuh"
#include "kv4.cuh"
#include "kv4_query.cuh"
#include "tc_dev.cuh"

#include <cuda_fp16.h>

namespace alice {
namespace {

constexpr uint32_t ROWS = KV4_PROMPT_ROWS, KEYS = 64, THREADS = 640;
// Registers by role; together what the launch has (65536 / 640 threads, down to a multiple of eight).
constexpr uint32_t REGS_ROWS = 136, REGS_OPERANDS = 72, REGS_REST = 64;
static_assert(256 * REGS_ROWS + 256 * REGS_OPERANDS + 128 * REGS_REST <= THREADS * (65536 / THREADS / 8 * 8), "");
constexpr uint32_t SCORES = 3;              // blocks whose scores or weights are in tensor memory
constexpr uint32_t RING = 4;                // blocks of keys as they lie in the pool
constexpr uint32_t GROUP = 4;               // blocks that share powers of two and whose sums add up in tensor memory
constexpr uint32_t SLOTS = 4;               // groups whose powers of two are there
constexpr int KERR_ATTN_WAIT = 9;           // a wait inside the tensor-core attention
constexpr float ROOM = 8.0f, LIFT = 7.0f;   // as in csrc/kv4_attn.cu
constexpr uint32_t NEVER = 0xffffffffu;

template <int NB>
struct Lay {
    // An operand: 64 columns of 64 keys a box; the values' boxes, a box for what codes are less than the numbers, the remainders' boxes.
    static constexpr uint32_t DIM = 32 * NB, BOXES = DIM / 64, BOX = KEYS * 128, BASE = BOXES * BOX, LEFT = BASE + BOX, OPERAND = LEFT + BASE;
    static constexpr uint32_t SUMS = SCORES * KEYS, QUERIES = SUMS + DIM + 16, TMEM = 512;      // columns: scores and weights, sums (and those of the bases), queries
    static_assert(QUERIES + DIM + 8 <= TMEM, "");
    static_assert(SUMS + DIM + 16 == QUERIES, "");
    static constexpr uint32_t TILE = kv4_tile_bytes(DIM);
    static constexpr uint32_t K = 0, V = 2 * OPERAND, TILES = 4 * OPERAND;                 // in shared memory; two operands each
    static constexpr uint32_t PLACE = V;                                                   // of the queries on their way to tensor memory
    static_assert(ROWS * DIM * 4 <= 2 * OPERAND, "");
    struct Smem {
        alignas(8) uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[SCORES], p_full[SCORES], p_empty[SCORES], o_empty, done[2];
        uint64_t came[RING], taken[RING], seen[SLOTS], over[SLOTS];                        // a block of the ring: is there, free; a group: looked over, over
        uint32_t tmem;
        float to[SLOTS][2], from[SLOTS][2];                                                // keys' and values' power of two, and its inverse
        uint32_t k_nan, v_nan[NB];                                                         // first positions
        float ref[ROWS], l[ROWS], top[2][2][ROWS];                                         // largest score of either half of the keys, blocks in turn
        float factor[ROWS], q_sum[ROWS][NB];
    };
    static constexpr size_t BYTES = sizeof(Smem) + 1024 + TILES + RING * 4 * TILE;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }
// f16 x f16 -> f32, M x N
__host__ __device__ constexpr uint32_t f16_desc(uint32_t m, uint32_t n, bool b_rows_k) { return (1u << 4) | ((uint32_t)b_rows_k << 16) | ((n / 8) << 17) | ((m / 16) << 24); }
__device__ __forceinline__ void pair_of(float a, float b, uint32_t& value, uint32_t& left) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    value = half2_bits(h); left = half2_bits(__floats2half2_rn(a - f.x, b - f.y));
}
__device__ __forceinline__ void cluster_sync() { asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t there(uint32_t a, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
    return r;
}
__device__ __forceinline__ float4 far_f4(uint32_t a) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t far_u32(uint32_t a) { uint32_t v; asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory"); return v; }
__device__ __forceinline__ float far_f32(uint32_t a) { return __uint_as_float(far_u32(a)); }
// A warp waits where it is blocks ahead: asleep between its questions, which would take issue slots from those that work.
__device__ __forceinline__ bool warp_rests(uint32_t bar, uint32_t parity) {
    const long long t0 = clock64();
    while (!__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) {
        __nanosleep(200);
        if (__any_sync(0xffffffffu, clock64() - t0 > WAIT_CYCLE_LIMIT)) return false;
    }
    return true;
}
// four lanes' or warps' arrivals in one
__device__ __forceinline__ void warp_arrive(uint32_t bar) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}
__device__ __forceinline__ void tmem_put8(uint32_t addr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::
          "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_ld8(float (&v)[8], uint32_t addr) {
    uint32_t r[8];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\ntcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(addr) : "memory");
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void sts16(uint32_t a, __half h) { asm volatile("st.shared.u16 [%0], %1;" ::"r"(a), "h"(__half_as_ushort(h)) : "memory"); }
__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
// The place of 8 columns (a 16-byte piece) of a row of a box.
__device__ __forceinline__ uint32_t piece_at(uint32_t row, uint32_t piece) { return row * 128 + ((piece ^ (row & 7)) << 4); }

}  // namespace

// grid (key / value heads of jobs, 1, parts of the keys), clusters along z.
template <int NB>
__global__ void __launch_bounds__(THREADS, 1) kv4_prompt_kernel(const __grid_constant__ Kv4AttnArgs a) {
    using L = Lay<NB>;
    constexpr uint32_t DIM = L::DIM, F4 = DIM / 4;
    extern __shared__ uint8_t raw[];
    auto& sh = *reinterpret_cast<typename L::Smem*>(raw);
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, part = blockIdx.z, parts = gridDim.z;
    const uint32_t job = blockIdx.x / a.shape.kv_heads, head = blockIdx.x - job * a.shape.kv_heads;      // all heads of the longest job go first
    const uint32_t smem = (smem_u32(raw) + (uint32_t)sizeof(typename L::Smem) + 1023u) & ~1023u;
    auto bar = [](uint64_t& b) { return smem_u32(&b); };
    if (tid == 0) {
        mbar_init(bar(sh.q_full), 8);
        for (int i = 0; i < 2; i++) {
            mbar_init(bar(sh.k_full[i]), 4); mbar_init(bar(sh.v_full[i]), 4); mbar_init(bar(sh.k_empty[i]), 1); mbar_init(bar(sh.v_empty[i]), 1);
            mbar_init(bar(sh.done[i]), 1);
        }
        for (uint32_t i = 0; i < SCORES; i++) { mbar_init(bar(sh.s_full[i]), 1); mbar_init(bar(sh.p_full[i]), 8); mbar_init(bar(sh.p_empty[i]), 1); }
        mbar_init(bar(sh.o_empty), 8);
        for (uint32_t i = 0; i < RING; i++) { mbar_init(bar(sh.came[i]), 1); mbar_init(bar(sh.taken[i]), 8); }
        for (uint32_t i = 0; i < SLOTS; i++) { mbar_init(bar(sh.seen[i]), 1); mbar_init(bar(sh.over[i]), 8); }
        mbar_fence_init();
        fence_proxy_async();
        sh.k_nan = NEVER;
        for (int b = 0; b < NB; b++) sh.v_nan[b] = NEVER;
    }
    if (warp == 16) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "n"(L::TMEM) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = sh.tmem;
    pdl_launch_dependents();      // not before the tensor memory is had: a later kernel's CTA could hold it and wait for this one
    pdl_wait();

    const Kv4Head hd = *a.plan.head;
    Kv4Job jb = a.plan.job[job];      // beside the head: not more than the plan has room for
    const bool here = kv4_fits(hd, a) && job < hd.prompt_jobs;
    if (!here) jb = Kv4Job{};
    const uint32_t keys = here ? jb.past + (jb.row + jb.rows - 1) / a.group + 1 : 0, blocks = (keys + KEYS - 1) / KEYS;
    const uint32_t b0 = blocks * part / parts, n = blocks * (part + 1) / parts - b0;

    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_ROWS));
        // ---- rows, a lane each of two warps: queries, the weights of half of the keys each, the sums of half of the dims ----
        constexpr uint32_t OWN = DIM / 2;
        const uint32_t quarter = warp & 3, hf = warp >> 2, row = quarter * 32 + lane, lane_at = tmem + ((quarter * 32) << 16);
        const uint32_t see = here && row < jb.rows ? jb.past + (jb.row + row) / a.group + 1 : 0;
        auto both = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory"); };      // the warps of a row meet, whatever has become of their waits
        float factor = 0;
        if (n) {
            // A row's dims lie 4 a lane to be read, rotated and cut into pairs, and go through shared memory into the lane of the row.
            constexpr uint32_t PER = DIM / 4, CH = 16 * DIM / 128, AT_ONCE = 4;
            const uint32_t place = smem + L::PLACE + quarter * 32 * DIM * 4, dim0 = lane % PER * 4;
            float4 x[CH];
            uint32_t of[CH];       // row of the rotation table
            // rows one after the other (of 64 dims every other): token and head without a division each; those behind the last are the last
            const uint32_t last = jb.row + jb.rows - 1, r0 = min(jb.row + quarter * 32 + hf * 16 + lane / PER, last);
            uint32_t r = r0, tok = r0 / a.group, of_group = r0 - tok * a.group;
#pragma unroll
            for (uint32_t c = 0; c < CH; c++) {
                const uint32_t at_tok = jb.first + tok;
                x[c] = *reinterpret_cast<const float4*>(a.q + at_tok * a.q_ld + (size_t)(head * a.group + of_group) * DIM + dim0);
                of[c] = a.rope.by_token ? at_tok : jb.past + tok;
#pragma unroll
                for (uint32_t k = 0; k < 128 / DIM; k++)
                    if (r < last) {
                        r++;
                        if (++of_group == a.group) { of_group = 0; tok++; }
                    }
            }
            if (a.rope.dims) {
                const uint32_t half = a.rope.dims / 2, turn_at = dim0 >= a.rope.dims ? 0 : a.rope.neox ? 2 * (dim0 < half ? dim0 : dim0 - half) : dim0;
#pragma unroll
                for (uint32_t c0 = 0; c0 < CH; c0 += AT_ONCE) {
                    Turn w[AT_ONCE];       // without a branch between the loads
#pragma unroll
                    for (uint32_t c = 0; c < AT_ONCE; c++) {
                        const float* const turn = a.rope.table + (size_t)of[c0 + c] * a.rope.dims + turn_at;
                        w[c].a = *reinterpret_cast<const float4*>(turn);
                        w[c].b = *reinterpret_cast<const float4*>(turn + (a.rope.neox ? 4 : 0));
                    }
#pragma unroll
                    for (uint32_t c = 0; c < AT_ONCE; c++) { const float4 one[1] = {x[c0 + c]}; x[c0 + c] = rotated4(one, 0, dim0, w[c], a.rope); }
                }
            }
#pragma unroll
            for (uint32_t c = 0; c < CH; c++) {
                const uint32_t own = hf * 16 + c * (128 / DIM) + lane / PER;
                const float f = quarter * 32 + own < jb.rows ? a.scale : 0.0f;
                const float v[4] = {x[c].x * f, x[c].y * f, x[c].z * f, x[c].w * f};
                float top = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
                if constexpr (PER == 32) top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));      // of numbers without a sign
                else {
#pragma unroll
                    for (uint32_t o = 1; o < PER; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                }
                int e2 = (int)((__float_as_uint(top) >> 23) & 0xff) - 127 - 9;     // the largest into 2^9 .. 2^10
                e2 = min(max(e2, -100), 120);
                const float down = pow2(-e2);
                uint32_t hi[2], lo[2];
                pair_of(v[0] * down, v[1] * down, hi[0], lo[0]);
                pair_of(v[2] * down, v[3] * down, hi[1], lo[1]);
                // 16-byte pieces of a row in an order that lets the rows' lanes read theirs side by side
                const uint32_t to = place + own * DIM * 4, piece = dim0 / 8, in = dim0 % 8 * 2;
                asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(to + ((piece ^ (own & 7)) << 4) + in), "r"(hi[0]), "r"(hi[1]) : "memory");
                asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(to + ((piece + DIM / 8 ^ (own & 7)) << 4) + in), "r"(lo[0]), "r"(lo[1]) : "memory");
                float sum = (v[0] + v[1] + v[2] + v[3]) * down;
#pragma unroll
                for (uint32_t o = 1; o < 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                if (lane % 8 == 0) sh.q_sum[quarter * 32 + own][dim0 / 32] = sum;
                if (dim0 == 0) sh.factor[quarter * 32 + own] = pow2(e2) * 1.44269504088896341f;
            }
            both();
            factor = sh.factor[row];
#pragma unroll
            for (uint32_t c = 0; c < OWN; c += 16) {       // one warp the values, one the remainders
                uint32_t w[16];
#pragma unroll
                for (uint32_t i = 0; i < 4; i++) {      // in the order of a word's unpacked codes: 0 4 1 5 2 6 3 7
                    const uint4 v = lds128(place + lane * DIM * 4 + ((hf * OWN / 4 + c / 4 + i ^ (lane & 7)) << 4));
                    w[4 * i] = __byte_perm(v.x, v.z, 0x5410); w[4 * i + 1] = __byte_perm(v.x, v.z, 0x7632);
                    w[4 * i + 2] = __byte_perm(v.y, v.w, 0x5410); w[4 * i + 3] = __byte_perm(v.y, v.w, 0x7632);
                }
                tmem_put16(lane_at + L::QUERIES + hf * OWN + c, w);
            }
            if (hf == 0) {       // sums of a block's queries, against the bases: values, values, remainders
                uint32_t w[8] = {};
#pragma unroll
                for (int b = 0; b < NB; b += 2) pair_of(sh.q_sum[row][b], sh.q_sum[row][b + 1], w[b / 2], w[4 + b / 2]);
                w[2] = w[0]; w[3] = w[1];
                tmem_put8(lane_at + L::QUERIES + DIM, w);
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            warp_arrive(bar(sh.q_full));
        }
        float sums[OWN], base[NB / 2], l = 0, ref = -INFINITY;      // weighted codes, weighted bases; of weights
#pragma unroll
        for (uint32_t c = 0; c < OWN; c++) sums[c] = 0;
#pragma unroll
        for (int b = 0; b < NB / 2; b++) base[b] = 0;
        const uint32_t all_see = here ? jb.past + jb.row / a.group + 1 : 0;      // keys that every row sees
        bool ok = true;
        float carried = 1.0f;          // what the reference's last move makes of the sums before it
        // the products of the block before the one at (place, turn) are over
        auto behind = [&](uint32_t place, uint32_t turn) { return warp_wait(bar(sh.p_empty[place ? place - 1 : SCORES - 1]), place ? turn : turn ^ 1); };
        // the sums of group g join the row's
        auto drain = [&](uint32_t g) {
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const float f = carried * sh.from[g % SLOTS][1];
#pragma unroll
            for (uint32_t c = 0; c < OWN; c += 32) {
                float v[32];
                tmem_ld32(v, lane_at + L::SUMS + hf * OWN + c);
#pragma unroll
                for (int i = 0; i < 32; i++) sums[c + i] = fmaf(v[i], f, sums[c + i]);
            }
            uint32_t v[16];
            tmem_get16(v, lane_at + L::SUMS + DIM);
            tmem_got16(v);
            auto sum_of = [&](int b) { return __uint_as_float(v[b]) + __uint_as_float(v[4 + b]); };
#pragma unroll
            for (int b = 0; b < NB / 2; b++) base[b] = fmaf(hf ? sum_of(NB / 2 + b) : sum_of(b), f, base[b]);
            l = fmaf(__uint_as_float(v[8]), carried, l);
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) { mbar_arrive(bar(sh.o_empty)); mbar_arrive(bar(sh.over[g % SLOTS])); }
        };
        uint32_t place_j = 0, turn_j = 0;      // j % SCORES, j / SCORES & 1
        for (uint32_t j = 0; j < n; j++) {
            ok = ok && warp_wait(bar(sh.s_full[place_j]), turn_j);
            const uint32_t at = lane_at + place_j * KEYS + hf * 32, key0 = (b0 + j) * KEYS + hf * 32;
            const float f = factor * sh.from[j / GROUP % SLOTS][0];
            float s[32];
            if (ok) {
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                tmem_ld32(s, at);
                const int left = (int)see - (int)key0;       // of these keys the row sees
                if (key0 + 32 > all_see) {
#pragma unroll
                    for (int i = 0; i < 32; i++) if (i >= left) s[i] = -INFINITY;
                }
                float most[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                for (int i = 4; i < 32; i++) most[i % 4] = fmaxf(most[i % 4], s[i]);
                sh.top[j & 1][hf][row] = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
            }
            both();
            if (!ok) continue;
            const float m = fmaxf(sh.top[j & 1][0][row], sh.top[j & 1][1][row]);
            carried = 1.0f;
            if (__any_sync(0xffffffffu, m * f > ref + ROOM)) {
                const float next = m * f > ref + ROOM ? m * f : ref;
                carried = next == ref ? 1.0f : ex2(ref - next);
                ref = next;
                l *= carried;
#pragma unroll
                for (uint32_t c = 0; c < OWN; c++) sums[c] *= carried;
#pragma unroll
                for (int b = 0; b < NB / 2; b++) base[b] *= carried;
                if (j % GROUP) {       // and those in tensor memory
                    if (!(ok = behind(place_j, turn_j))) continue;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
                    for (uint32_t c = 0; c <= OWN; c += 16) {
                        if (c == OWN && hf) break;
                        const uint32_t sums_at = lane_at + L::SUMS + (c == OWN ? DIM : hf * OWN + c);
                        uint32_t v[16];
                        tmem_get16(v, sums_at);
                        tmem_got16(v);
#pragma unroll
                        for (int i = 0; i < 16; i++) v[i] = __float_as_uint(__uint_as_float(v[i]) * carried);
                        tmem_put16(sums_at, v);
                    }
                }
            }
            const float lift = ref == -INFINITY ? 0.0f : LIFT - ref;      // a row that has seen nothing yet: its scores stay -inf
            uint32_t out[32];
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const float p0 = ex2(fmaf(s[2 * i], f, lift)), p1 = ex2(fmaf(s[2 * i + 1], f, lift));
                pair_of(p0, p1, out[i], out[16 + i]);
            }
            tmem_put32(at, out);
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            warp_arrive(bar(sh.p_full[place_j]));
            if (j && j % GROUP == 0 && (ok = behind(place_j, turn_j))) drain(j / GROUP - 1);
            if (++place_j == SCORES) { place_j = 0; turn_j ^= 1; }
        }
        carried = 1.0f;
        if (ok && n && (ok = behind(place_j, turn_j))) drain((n - 1) / GROUP);
        if (!ok && lane == 0) atomicCAS(a.status, 0, KERR_ATTN_WAIT);
        // the last products are over: the place of their operands is free
#pragma unroll
        for (uint32_t i = 0; i < F4 / 2; i++) {
            const uint32_t o = smem + (row * F4 + (hf * (F4 / 2) + i ^ (row & (F4 - 1)))) * 16, c = i / 2 * 8 + i % 2;      // columns in the order of unpacked codes
            const float x = base[i / 8];
            asm volatile("st.shared.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(o), "f"(sums[c] + x), "f"(sums[c + 2] + x), "f"(sums[c + 4] + x), "f"(sums[c + 6] + x) : "memory");
        }
        if (hf == 0) { sh.ref[row] = ref; sh.l[row] = l; }
    } else if (warp < 16) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_OPERANDS));
        // ---- operands: four warps keys, four warps values; (position, block of 32 dims) by thread ----
        constexpr int ITEMS = NB / 2;
        constexpr uint32_t STEP = KEYS / ITEMS;      // positions from one of a thread's items to the next
        const bool is_v = warp >= 12;
        const uint32_t t = tid & 127, pos = t / (8 * NB) * 8 + (t & 7), b = t >> 3 & (NB - 1), pr = kv4_row(pos % KV4_TILE);
        // Words of a row in an order of the row's own, so that neither these loads nor the stores of the operand's pieces meet in a bank: word i ^ turn, of
        // keys x -> w x in the field of four (a multiplication that plus x is one again).
        const uint32_t x = pos & 3, turn = is_v ? pos >> 1 & 3 : (x ^ x >> 1) << 1 & 2 | x >> 1;
        const uint32_t tile = smem + L::TILES + pos / KV4_TILE * L::TILE, codes_at = tile + (is_v ? kv4_v_codes(DIM) + pos % KV4_TILE * (DIM / 2) + b * 2 : pr * (DIM / 2) + b * 4);
        const uint32_t scales_at = tile + (is_v ? kv4_v_scales(DIM) : kv4_k_scales(DIM)) + pr * (4 * NB) + b * 2, operands = smem + (is_v ? L::V : L::K);
        bool ok = true;
        if (is_v && n) ok = warp_wait(bar(sh.q_full), 0);      // the queries have left the place
        // The columns that the bases do not fill are zero once and for all (of values the ninth is one: the sum of the weights): of both operands, the rows that this
        // warp writes.
        if (ok) {
            const uint32_t row = NB == 4 ? t / 32 * 8 + (lane & 7) + (lane >> 3 & 1) * 32 : t / 32 * 16 + (lane & 15);
#pragma unroll
            for (int i = 0; i < 2; i++) sts128(operands + i * L::OPERAND + L::BASE + piece_at(row, lane >> 4), is_v && lane >> 4 ? 0x3c00 : 0, 0, 0, 0);
            __syncwarp();
        }
        for (uint32_t j = 0; j < n && ok; j++) {
            const uint32_t st = j & 1, at = j % RING * 4 * L::TILE, slot = j / GROUP % SLOTS;
            ok = (j % GROUP || warp_wait(bar(sh.seen[slot]), j / GROUP / SLOTS & 1)) && warp_wait(bar(sh.came[j % RING]), (j / RING) & 1);
            if (!ok) break;
            uint32_t codes[ITEMS][4], d16[ITEMS], m16[ITEMS];
#pragma unroll
            for (int h = 0; h < ITEMS; h++) {
                const uint32_t from = codes_at + at + h * (STEP / KV4_TILE) * L::TILE, scales = scales_at + at + h * (STEP / KV4_TILE) * L::TILE;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t o = from + (i ^ turn) * (NB * 4);
                    codes[h][i] = is_v ? lds16(o) | lds16(o + NB * 2) << 16 : lds32(o);
                }
                d16[h] = lds16(scales); m16[h] = lds16(scales + 2 * NB);
                if ((b0 + j) * KEYS + pos + h * STEP >= keys) d16[h] = m16[h] = 0;      // what lies behind the last key is anything
            }
            const float to = sh.to[slot][is_v];
            warp_arrive(bar(sh.taken[j % RING]));
            if (!(ok = warp_wait(bar(is_v ? sh.v_empty[st] : sh.k_empty[st]), ((j >> 1) & 1) ^ 1))) break;
            // A row's 32 dims: step * (code - 8) as values and remainders (of 15 bits: exact), minimum + 8 * step beside them
#pragma unroll
            for (int h = 0; h < ITEMS; h++) {
                float d = f16_bits_to_f32(d16[h]), m = f16_bits_to_f32(m16[h]);
                if (m != m) d = m = 0;
                const __half2 step = __half2half2(__float2half_rn(d * to));
                const uint32_t row = operands + st * L::OPERAND + h * STEP * 128;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const Codes c = unpack<8>(codes[h][i]);
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const __half2 v = __hmul2(bits_half2(c.v[k]), step);
                        hi[k] = half2_bits(v); lo[k] = half2_bits(__hfma2(bits_half2(c.v[k]), step, __hneg2(v)));
                    }
                    const uint32_t o = row + b / 2 * L::BOX + piece_at(pos, (b & 1) * 4 + (i ^ turn));
                    sts128(o, hi[0], hi[1], hi[2], hi[3]);
                    sts128(o + L::LEFT, lo[0], lo[1], lo[2], lo[3]);
                }
                const float base = fmaf(8.0f, d, m) * to;
                const __half v = __float2half_rn(base);
                const uint32_t o = row + L::BASE + b * 2;
                sts16(o + piece_at(pos, 0), v);
                sts16(o + piece_at(pos, 0) + 8, __float2half_rn(base - __half2float(v)));
                if (!is_v) sts16(o + piece_at(pos, 1), v);
            }
            fence_proxy_async();
            warp_arrive(bar(is_v ? sh.v_full[st] : sh.k_full[st]));
        }
        if (!ok && lane == 0) atomicCAS(a.status, 0, KERR_ATTN_WAIT);
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_REST));
        bool ok = true;
        // ---- products: two warps, so that one's waits are filled with the other's ----
        if (warp == 16 && n) {
            ok = warp_wait(bar(sh.q_full), 0);
            constexpr uint32_t desc = f16_desc(ROWS, KEYS, false);
            uint32_t place_j = 0, turn_j = 0;
            for (uint32_t j = 0; j < n && ok; j++) {
                ok = warp_wait(bar(sh.p_empty[place_j]), turn_j ^ 1) && warp_wait(bar(sh.k_full[j & 1]), (j >> 1) & 1);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (elect_lane()) {
                    const uint32_t kv = smem + L::K + (j & 1) * L::OPERAND, to = tmem + place_j * KEYS, q = tmem + L::QUERIES;
                    auto keys16 = [&](uint32_t from, uint32_t kk) { return smem_desc(kv + from + kk / 4 * L::BOX) + 2 * (kk % 4); };
                    // small products first: fewer steps of a sum that is large already
#pragma unroll
                    for (uint32_t kk = 0; kk < DIM / 16; kk++) {
                        mma_f16_ta(to, q + kk * 8, keys16(L::LEFT, kk), desc, kk > 0);
                        mma_f16_ta(to, q + DIM / 2 + kk * 8, keys16(0, kk), desc, true);
                    }
#pragma unroll
                    for (uint32_t kk = 0; kk < DIM / 16; kk++) mma_f16_ta(to, q + kk * 8, keys16(0, kk), desc, true);
                    mma_f16_ta(to, q + DIM, smem_desc(kv + L::BASE), desc, true);
                    mma_commit(bar(sh.s_full[place_j]));
                    mma_commit(bar(sh.k_empty[j & 1]));
                }
                __syncwarp();
                if (++place_j == SCORES) { place_j = 0; turn_j ^= 1; }
            }
            if (elect_lane()) mma_commit(bar(sh.done[0]));
            __syncwarp();
            ok = warp_wait(bar(sh.done[0]), 0) && ok;      // nothing of it runs any more
        } else if (warp == 19 && n) {
            constexpr uint32_t desc = f16_desc(ROWS, DIM, true), both_desc = f16_desc(ROWS, DIM + 16, true);
            uint32_t place_j = 0, turn_j = 0;
            for (uint32_t j = 0; j < n; j++) {
                ok = warp_wait(bar(sh.v_full[j & 1]), (j >> 1) & 1) && (j % GROUP || warp_wait(bar(sh.o_empty), (j / GROUP & 1) ^ 1)) && warp_wait(bar(sh.p_full[place_j]), turn_j);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (elect_lane()) {
                    const uint32_t va = smem + L::V + (j & 1) * L::OPERAND, pa = tmem + place_j * KEYS, to = tmem + L::SUMS;
                    auto weights = [&](uint32_t c) { return pa + c / 2 * 32 + c % 2 * 8; };      // of sixteen keys: values; remainders 16 columns on
                    auto keys16 = [&](uint32_t from, uint32_t c) { return smem_desc_n(va + from + c * 16 * 128, L::BOX); };
#pragma unroll
                    for (uint32_t c = 0; c < KEYS / 16; c++) mma_f16_ta(to, weights(c) + 16, keys16(0, c), both_desc, c > 0 || j % GROUP);
#pragma unroll
                    for (uint32_t c = 0; c < KEYS / 16; c++) mma_f16_ta(to, weights(c), keys16(L::LEFT, c), desc, true);
#pragma unroll
                    for (uint32_t c = 0; c < KEYS / 16; c++) mma_f16_ta(to, weights(c), keys16(0, c), both_desc, true);
                    mma_commit(bar(sh.v_empty[j & 1]));
                    mma_commit(bar(sh.p_empty[place_j]));
                }
                __syncwarp();
                if (++place_j == SCORES) { place_j = 0; turn_j ^= 1; }
            }
            if (elect_lane()) mma_commit(bar(sh.done[1]));
            __syncwarp();
            ok = warp_wait(bar(sh.done[1]), 0) && ok;
        } else if (warp == 17) {
            // ---- the ring: a block is four tiles, a lane each ----
            const uint32_t per_page = a.shape.tiles();
            uint32_t j = 0;
            for (; j < n; j++) {
                const uint32_t tile = (b0 + j) * 4 + lane, s = j % RING;
                const bool mine = lane < 4 && tile * KV4_TILE < keys;
                const uint32_t pg = mine ? tile / per_page : 0, page = mine ? a.plan.table[(size_t)jb.seq * a.plan.table_ld + pg] : 0;
                const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, mine)) * L::TILE;
                if (!(ok = warp_rests(bar(sh.taken[s]), ((j / RING) & 1) ^ 1))) break;
                if (lane == 0) mbar_arrive_expect_tx(bar(sh.came[s]), bytes);
                __syncwarp();
                if (mine)
                    bulk_g2s(smem + L::TILES + (s * 4 + lane) * L::TILE, a.pool + (((size_t)page * a.shape.kv_heads + head) * per_page + (tile - pg * per_page)) * L::TILE, L::TILE, bar(sh.came[s]));
                __syncwarp();
            }
            for (uint32_t i = j < RING ? 0 : j - RING; i < j; i++) ok = warp_wait(bar(sh.came[i % RING]), (i / RING) & 1) && ok;      // no copy is on its way any more
        } else if (warp == 18) {
            // ---- the keys' and the values' largest magnitude in a group, and their first NaN: scales of 64 rows a block from the pool, ahead of the ring ----
            const uint32_t per_page = a.shape.tiles(), which = lane >> 4, row = lane & 15;      // keys, values; a tile at a time
            for (uint32_t g = 0; g * GROUP < n; g++) {
                constexpr uint32_t AT_ONCE = GROUP * 2;
                const uint32_t tile0 = (b0 + g * GROUP) * 4, tiles = min(GROUP * 4, (keys + KV4_TILE - 1) / KV4_TILE - tile0), end = min(GROUP, n - g * GROUP) * 4;
                const uint32_t own = tile0 + min(row, tiles - 1), pg = own / per_page;
                const uint32_t own_at = a.plan.table[(size_t)jb.seq * a.plan.table_ld + pg] * a.shape.kv_heads * per_page + head * per_page + (own - pg * per_page);
                float most = 0;
#pragma unroll 1
                for (uint32_t i0 = 0; i0 < GROUP * 4; i0 += AT_ONCE) {
                    uint2 d[AT_ONCE], m[AT_ONCE];        // of a row (of 64 dims in one word each)
#pragma unroll
                    for (uint32_t i = 0; i < AT_ONCE; i++) {
                        const uint32_t at = __shfl_sync(0xffffffffu, own_at, i0 + i);
                        const uint8_t* const p = a.pool + (size_t)at * L::TILE + (which ? kv4_v_scales(DIM) : kv4_k_scales(DIM)) + row * (4 * NB);
                        if constexpr (NB == 4) { const uint4 v = *reinterpret_cast<const uint4*>(p); d[i] = make_uint2(v.x, v.y); m[i] = make_uint2(v.z, v.w); }
                        else { const uint2 v = *reinterpret_cast<const uint2*>(p); d[i] = make_uint2(v.x, 0); m[i] = make_uint2(v.y, 0); }
                    }
#pragma unroll
                    for (uint32_t i = 0; i < AT_ONCE; i++) {
                        const uint32_t key = (tile0 + i0 + i) * KV4_TILE + ((row & 8) | (row & 1) << 2 | (row >> 1 & 3));      // the position whose scales lie in this row
                        if (i0 + i >= min(tiles, end) || key >= keys) continue;
                        auto two = [&](uint32_t dd, uint32_t mm, int b) {
                            const float2 df = __half22float2(bits_half2(dd)), mf = __half22float2(bits_half2(mm));
#pragma unroll
                            for (int k = 0; k < 2; k++) {
                                const float dk = k ? df.y : df.x, mk = k ? mf.y : mf.x;
                                if (mk != mk) atomicMin(which ? &sh.v_nan[b + k] : &sh.k_nan, key);
                                else most = fmaxf(most, fmaxf(8.0f * dk, fabsf(fmaf(8.0f, dk, mk))));
                            }
                        };
                        two(d[i].x, m[i].x, 0);
                        if constexpr (NB == 4) two(d[i].y, m[i].y, 2);
                    }
                }
#pragma unroll
                for (uint32_t o = 1; o < 16; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
                const uint32_t top = __float_as_uint(most);      // below 2^15 with this exponent: codes * step and base are as large at most
                const int e = top ? 14 - ((int)(top >> 23) - 127) : 0;
                if (!(ok = warp_rests(bar(sh.over[g % SLOTS]), (g / SLOTS & 1) ^ 1))) break;
                if (row == 0) { sh.to[g % SLOTS][which] = pow2(e); sh.from[g % SLOTS][which] = pow2(-e); }
                warp_arrive(bar(sh.seen[g % SLOTS]));
            }
        }
        if (!ok && lane == 0) atomicCAS(a.status, 0, KERR_ATTN_WAIT);
    }
    // ---- parts of the keys joined, out ----
    if (parts > 1) cluster_sync(); else __syncthreads();
    if (here) {
        const uint32_t rows_each = (ROWS + parts - 1) / parts;
        uint32_t k_nan = NEVER;
        for (uint32_t c = 0; c < parts; c++) k_nan = min(k_nan, far_u32(there(smem_u32(&sh.k_nan), c)));
        for (uint32_t i = tid; i < rows_each * F4; i += THREADS) {
            const uint32_t row = part * rows_each + i / F4, f4 = i % F4;
            if (row >= jb.rows) break;
            const uint32_t r = jb.row + row, tok = r / a.group, see = jb.past + tok + 1, mine = (row * F4 + (f4 ^ (row & (F4 - 1)))) * 16;
            float m = -INFINITY, sum = 0;
            uint32_t v_nan = NEVER;
            for (uint32_t c = 0; c < parts; c++) {
                m = fmaxf(m, far_f32(there(smem_u32(&sh.ref[row]), c)));
                v_nan = min(v_nan, far_u32(there(smem_u32(&sh.v_nan[f4 / 8]), c)));
            }
            float4 o = make_float4(0, 0, 0, 0);
            for (uint32_t c = 0; c < parts; c++) {
                const float ref = far_f32(there(smem_u32(&sh.ref[row]), c)), l = far_f32(there(smem_u32(&sh.l[row]), c));
                const float4 x = far_f4(there(smem + mine, c));
                const float f = ref == m ? 1.0f : ex2(ref - m);
                sum = fmaf(l, f, sum);
                o.x = fmaf(x.x, f, o.x); o.y = fmaf(x.y, f, o.y); o.z = fmaf(x.z, f, o.z); o.w = fmaf(x.w, f, o.w);
            }
            const float inv = see > k_nan || see > v_nan ? __uint_as_float(0x7fc00000u) : 1.0f / sum;
            *reinterpret_cast<float4*>(a.out + (size_t)(jb.first + tok) * a.out_ld + (size_t)(head * a.group + r - tok * a.group) * DIM + 4 * f4) =
                make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
        }
    }
    if (parts > 1) cluster_sync();      // what the others read stays until they have
    if (warp == 16) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(L::TMEM));
    }
}

namespace {
// Parts of the keys of a job (a cluster): those with which clusters side by side, one after the other, take the least time. A cluster's start and join are counted as
// eight blocks of keys of 2600 clocks (2048 tokens of 32 x 8 heads: the start is 14 to 18 thousand of a CTA's 95 thousand clocks).
uint32_t parts_of(uint32_t clusters, uint32_t blocks, const int (&at_once)[9]) {
    uint32_t best = 1;
    uint64_t least = ~0ull;
    for (uint32_t p = 1; p <= 8 && p <= blocks; p++) {
        if (at_once[p] <= 0) continue;
        const uint64_t t = ((uint64_t)clusters + at_once[p] - 1) / at_once[p] * (8 + (blocks + p - 1) / p);
        if (t < least) { least = t; best = p; }
    }
    return best;
}

template <int NB>
cudaError_t launch(const Kv4AttnArgs& a, cudaStream_t st, bool pdl) {
    using L = Lay<NB>;
    static int at_once[64][9] = {};      // clusters of .. CTAs that a device holds; [0]: known
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return err;
    if (dev >= 64) return cudaErrorInvalidDevice;
    constexpr size_t smem = L::BYTES > 120 * 1024 ? L::BYTES : 120 * 1024;      // one CTA an SM: each takes all of the tensor memory
    static_assert(smem <= 227 * 1024, "");
    cudaLaunchConfig_t lc = {}; cudaLaunchAttribute at[2];
    lc.blockDim = dim3(THREADS); lc.dynamicSmemBytes = smem; lc.stream = st;
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = at[0].val.clusterDim.y = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = at;
    if (!at_once[dev][0]) {
        err = cudaFuncSetAttribute(kv4_prompt_kernel<NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (err != cudaSuccess) return err;
        for (uint32_t p = 1; p <= 8; p++) {
            lc.gridDim = dim3(1, 1, p); at[0].val.clusterDim.z = p; lc.numAttrs = 1;
            if ((err = cudaOccupancyMaxActiveClusters(&at_once[dev][p], kv4_prompt_kernel<NB>, &lc)) != cudaSuccess) return err;
        }
        at_once[dev][0] = 1;
    }
    const uint32_t parts = parts_of(a.prompt_jobs * a.shape.kv_heads, (a.end + KEYS - 1) / KEYS, at_once[dev]);
    lc.gridDim = dim3(a.prompt_jobs * a.shape.kv_heads, 1, parts); at[0].val.clusterDim.z = parts; lc.numAttrs = pdl ? 2 : 1;
    return cudaLaunchKernelEx(&lc, kv4_prompt_kernel<NB>, a);
}
}  // namespace

cudaError_t launch_kv4_prompt(const Kv4AttnArgs& a, cudaStream_t st, bool pdl) {
    switch (a.shape.dim) {
        case 64: return launch<2>(a, st, pdl);
        case 128: return launch<4>(a, st, pdl);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace alice
