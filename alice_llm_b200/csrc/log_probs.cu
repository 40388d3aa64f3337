// Log probabilities, entropy, rank and the most probable tokens of rows of logits.
//
// With m the largest logit and s the sum of exp(x - m) over all others but that one:
//   log p(x) = (x - m) - log1p(s),   H = log1p(s) - w / (1 + s),   w = sum (x - m) exp(x - m)
// so that what is small beside the largest term is not lost where one token has nearly all the weight. Every partial sum, of a thread,
// a warp or a CTA, is a triple (m, s, w) in which the 1 of its own largest term is left out.
//
// One pass: a thread takes 16 logits at a time, splits them into their largest and the 15 others by minima and maxima and adds them to its
// triple. The alternatives come from the same registers: a bound that at least k of the threads' first maxima reach and few more is found by
// halving; logits above it go to a list in shared memory, later ones too, without a barrier, and now and then the list is put in order and
// the bound rises to its k-th. Should it overflow all the same (logits that keep rising), the part is listed again, 16 logits a thread
// and a barrier at a time. A row is cut among the CTAs of a cluster, as many as keep the chip busy, and joined through distributed shared memory: no scratch,
// nothing that calls or graphs could share, and the same order of sums at every call.
#include <algorithm>
#include <cmath>

#include "abi_internal.cuh"
#include "common.cuh"
#include "log_probs.cuh"
#include "rows.cuh"

namespace alice {

namespace {

// Logits in order as whole numbers, the lower index first among equals. 0: no logit.
__device__ __forceinline__ unsigned long long logit_key(float x, uint32_t i) {
    const uint32_t u = __float_as_uint(x + 0.0f);      // -0 as 0
    return (unsigned long long)(u & 0x80000000u ? ~u : u | 0x80000000u) << 32 | (0xffffffffu - i);
}
__device__ __forceinline__ float key_logit(unsigned long long k) {
    const uint32_t u = (uint32_t)(k >> 32);
    return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}

constexpr int THREADS = 256, WARPS = THREADS / 32, FOURS = 4, EACH = 4 * FOURS;      // a thread's logits at a time
constexpr uint32_t MAX_CLUSTER = 16;
// Entries of the list. A bound may be reached by as many threads as leave room for all their logits beside the alternatives so far.
constexpr uint32_t CAP = 1024, REACH = (CAP - LOGP_MAX_TOP) / EACH;
static_assert(MAX_CLUSTER * LOGP_MAX_TOP <= CAP && REACH >= LOGP_MAX_TOP, "");
constexpr float LEAST = -3.402823466e38f;

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float exp_of(float t) {     // t <= 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(t * 1.44269504088896341f));
    return y;
}
// Differences end at -200, whose exponential is 0: the term of a ruled-out token is 0 and not 0 times infinity.
__device__ __forceinline__ float diff(float x, float m) { return max_nan(x - m, -200.0f); }

struct Triple {
    float m, s, w;
    __device__ __forceinline__ void join(const Triple& o) {
        const float top = max_nan(m, o.m), ref = max_nan(top, LEAST);
        const bool first = m >= o.m;
        const float t = diff(first ? o.m : m, ref), f = exp_of(t), ls = (first ? o.s : s) + 1.0f, lw = first ? o.w : w;
        s = fmaf(f, ls, first ? s : o.s);
        w = fmaf(f, fmaf(t, ls, lw), first ? w : o.w);
        m = top;
    }
};
// Of the first N lanes: each of them has the whole.
template <int N>
__device__ __forceinline__ void join_lanes(Triple& me, uint32_t& count) {
#pragma unroll
    for (int o = N / 2; o > 0; o >>= 1) {
        Triple you;
        you.m = __shfl_xor_sync(0xffffffffu, me.m, o); you.s = __shfl_xor_sync(0xffffffffu, me.s, o); you.w = __shfl_xor_sync(0xffffffffu, me.w, o);
        count += __shfl_xor_sync(0xffffffffu, count, o);
        me.join(you);
    }
}
__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm("mov.u32 %0, %cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t cluster_size() { uint32_t r; asm("mov.u32 %0, %cluster_nctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t there(const void* p, uint32_t rank) {      // the same place in another CTA
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
    return r;
}
__device__ __forceinline__ float far_f32(uint32_t a) { float v; asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory"); return v; }
__device__ __forceinline__ uint32_t far_u32(uint32_t a) { uint32_t v; asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory"); return v; }
__device__ __forceinline__ unsigned long long far_u64(uint32_t a) { unsigned long long v; asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a) : "memory"); return v; }

struct Smem {
    Triple part[WARPS];
    uint32_t above[WARPS];
    Triple all;
    uint32_t all_above, listed;                      // logits above the target; entries of `top`
    uint32_t entering;                               // of `cand`
    unsigned long long bound;
    unsigned long long most[THREADS];                // the threads' largest
    unsigned long long top[LOGP_MAX_TOP];            // the list, the largest first
    unsigned long long cand[CAP];
};

// cand[0 .. n) in order: the first `want` of them to top. All threads, four to an entry; n and want are the CTA's.
__device__ __forceinline__ uint32_t put_in_order(Smem& sh, uint32_t n, uint32_t want) {
    const uint32_t q = threadIdx.x & 3;
    for (uint32_t i0 = 0; i0 < n; i0 += THREADS / 4) {
        const uint32_t i = i0 + threadIdx.x / 4;
        const unsigned long long k = i < n ? sh.cand[i] : 0ull;
        uint32_t before = 0;
#pragma unroll 4
        for (uint32_t j = q; j < n; j += 4) before += sh.cand[j] > k;
        before += __shfl_xor_sync(0xffffffffu, before, 1);
        before += __shfl_xor_sync(0xffffffffu, before, 2);
        if (i < n && q == 0 && before < want) sh.top[before] = k;
    }
    return min(n, want);
}

}  // namespace

// Measured: 1 row of 128256 without alternatives 4.8 us, with 5 9.8; 777 of 32000 without 24.0 (4.1 TB/s); 256 of 151643 with 20 50.2 (3.1 TB/s: comparisons with the
// bound and exponentials share the issue slots; without alternatives the loads bound it).
template <bool TOP>
__global__ void __launch_bounds__(THREADS, 4) log_probs_kernel(const __grid_constant__ LogProbArgs a) {
    __shared__ Smem sh;
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, parts = cluster_size(), part = cluster_rank();
    const size_t r = blockIdx.x / parts;
    // The row in pieces of four that lie on 16-byte boundaries; its first and last may hold less of it.
    const float* const row = a.x + r * a.ld;
    const uint32_t skip = (uint32_t)((reinterpret_cast<uintptr_t>(row) >> 2) & 3);
    const float4* const four = reinterpret_cast<const float4*>(row - skip);
    const uint32_t fours = (uint32_t)(((uint64_t)a.vocab + skip + 3) / 4), per = (fours + parts - 1) / parts, begin = min(part * per, fours), end = min(begin + per, fours);
    const uint32_t whole0 = skip ? 1 : 0, whole1 = min(end, (uint32_t)(((uint64_t)a.vocab + skip) / 4));      // pieces that are the row's own
    auto load = [&](float (&x)[EACH], uint32_t at) {
        // Without a look at every piece's ends: 256 rows of 151643 with 20 alternatives 56.6 -> 50.2 us, but 777 of 32000 without any 23.9 -> 25.7 (the code of
        // both ways stands between the loads and their use).
        if (TOP && at >= whole0 && at + FOURS * THREADS <= whole1) {
#pragma unroll
            for (int i = 0; i < FOURS; i++) {
                const float4 v = __ldcs(four + at + tid + i * THREADS);
                x[4 * i] = v.x; x[4 * i + 1] = v.y; x[4 * i + 2] = v.z; x[4 * i + 3] = v.w;
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < FOURS; i++) {
            const uint32_t p = at + i * THREADS + tid;
            float4 v = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            if (p < end) {
                const long long e = (long long)p * 4 - skip;
                if (e >= 0 && e + 4 <= (long long)a.vocab) v = __ldcs(four + p);
                else {
                    float* const f = &v.x;
#pragma unroll
                    for (int j = 0; j < 4; j++) if (e + j >= 0 && e + j < (long long)a.vocab) f[j] = __ldcs(row + (e + j));
                }
            }
            x[4 * i] = v.x; x[4 * i + 1] = v.y; x[4 * i + 2] = v.z; x[4 * i + 3] = v.w;
        }
    };
    float x[EACH], next[EACH];
    load(x, begin);
    const uint32_t t = a.target ? a.target[r] : 0u;
    const bool aimed = a.target && t < a.vocab;
    const float xt = aimed ? row[t] : INFINITY;
    if (tid == 0) { sh.listed = 0; sh.entering = 0; }
    if (TOP) __syncthreads();

    Triple me{-INFINITY, 0, 0};
    uint32_t above = 0;
    unsigned long long from = 0;          // what is larger enters the list
    auto key = [&](int i, uint32_t at) {          // what is past the row is no logit
        const long long e = (long long)(at + (i >> 2) * THREADS + tid) * 4 - skip + (i & 3);
        return at + (i >> 2) * THREADS + tid < end && e >= 0 && e < (long long)a.vocab ? logit_key(x[i], (uint32_t)e) : 0ull;
    };
    // the list's first, in order, and nothing else of it
    auto compact = [&](uint32_t n) {
        put_in_order(sh, n, a.top);
        __syncthreads();
        if (tid < a.top) sh.cand[tid] = sh.top[tid];
        if (tid == 0) sh.entering = a.top;
        from = sh.top[a.top - 1];
    };
    // 16 logits a thread into the list, all threads together
    auto enter = [&](uint32_t at, float big) {
            const bool reach = from == 0 || big >= key_logit(from);
            const uint32_t over = __syncthreads_count(reach);
            if (over) {
                uint32_t n = sh.entering;
                if (n + over * EACH > CAP) {
                    if (n > a.top) { compact(n); n = a.top; }
                    if (over > REACH) {
                        sh.most[tid] = logit_key(big, 0);
                        __syncthreads();
                        if (warp == 0) {         // by the bits in which they differ, from the highest
                            uint32_t k[THREADS / 32], lo = 0xffffffffu, hi = 0;
#pragma unroll
                            for (int i = 0; i < THREADS / 32; i++) { k[i] = (uint32_t)(sh.most[lane + 32 * i] >> 32); lo = min(lo, k[i]); hi = max(hi, k[i]); }
                            lo = __reduce_min_sync(0xffffffffu, lo); hi = __reduce_max_sync(0xffffffffu, hi);
                            const int bits = 32 - __clz(lo ^ hi);
                            uint32_t found = bits == 32 ? 0u : hi >> bits << bits, at_least = THREADS;
                            for (int bit = bits - 1; bit >= 0 && at_least > a.top + a.top / 4 + 1; bit--) {
                                const uint32_t trial = found | 1u << bit;
                                uint32_t c = 0;
#pragma unroll
                                for (int i = 0; i < THREADS / 32; i++) c += k[i] >= trial;
                                c = __reduce_add_sync(0xffffffffu, c);
                                if (c >= a.top) { found = trial; at_least = c; }
                            }
                            if (lane == 0) sh.bound = at_least <= REACH ? (unsigned long long)found << 32 : ~0ull;
                        }
                        __syncthreads();
                        unsigned long long bound = sh.bound;
                        if (bound == ~0ull) {    // too many that are equal: by their places too
                            unsigned long long mine = 0;
#pragma unroll
                            for (int i = 0; i < EACH; i++) { const unsigned long long k = key(i, at); mine = k > mine ? k : mine; }
                            sh.most[tid] = mine;
                            __syncthreads();
                            if (warp == 0) {
                                unsigned long long found = 0;
                                for (int bit = 63; bit >= 0; bit--) {
                                    const unsigned long long trial = found | 1ull << bit;
                                    uint32_t c = 0;
                                    for (int i = 0; i < THREADS / 32; i++) c += sh.most[lane + 32 * i] >= trial;
                                    if (__reduce_add_sync(0xffffffffu, c) >= a.top) found = trial;
                                }
                                if (lane == 0) sh.bound = found;
                            }
                            __syncthreads();
                            bound = sh.bound;    // the top-th largest, or 0 where there are not so many
                        }
                        if (bound > from) from = bound - 1;
                    }
                }
                __syncthreads();
                const float least = from == 0 ? -INFINITY : key_logit(from);
                if (big >= least) {
#pragma unroll
                    for (int i = 0; i < EACH; i++)
                        if (x[i] >= least) { const unsigned long long k = key(i, at); if (k > from) sh.cand[atomicAdd(&sh.entering, 1u)] = k; }
                }
            }
    };
    uint32_t round = 0;
    for (uint32_t at = begin; at < end; at += FOURS * THREADS) {
        if (at + FOURS * THREADS < end) load(next, at + FOURS * THREADS);
        // ---- the largest, and the others ----
        float big = x[0], other[EACH];
#pragma unroll
        for (int i = 1; i < EACH; i++) {
            other[i] = fminf(big, x[i]);
            big = max_nan(big, x[i]);
        }
#pragma unroll
        for (int i = 0; i < EACH; i++) above += x[i] > xt;
        {
            const float top = max_nan(me.m, big), ref = max_nan(top, LEAST);
            const bool moved = me.m < top;
            const float d = diff(moved ? me.m : big, ref), f = exp_of(d);      // of the two largest, the lesser
            if (at == begin) me.s = me.w = 0;                                    // there is only one
            else if (moved) { me.w = f * fmaf(d, me.s + 1.0f, me.w); me.s = f * (me.s + 1.0f); }
            else { me.s += f; me.w = fmaf(f, d, me.w); }
            float s = 0, w = 0;
#pragma unroll
            for (int i = 1; i < EACH; i++) {
                const float z = diff(other[i], ref), e = exp_of(z);
                s += e;
                w = fmaf(e, z, w);
            }
            me.s += s; me.w += w; me.m = top;
        }
        // ---- the list ----
        if (TOP) {
            if (at == begin) enter(at, big);
            else {
                if ((++round & (round - 1)) == 0 && round > 1) {      // 2, 4, 8, ...: as many logits again as there were. The same for all threads
                    __syncthreads();
                    const uint32_t n = sh.entering;
                    if (n > a.top && n <= CAP) compact(n);
                    __syncthreads();
                }
                const float least = from == 0 ? -INFINITY : key_logit(from);
                if (big >= least) {
#pragma unroll
                    for (int i = 0; i < EACH; i++)
                        if (x[i] >= least) {
                            const unsigned long long k = key(i, at);
                            if (k > from) { const uint32_t to = atomicAdd(&sh.entering, 1u); if (to < CAP) sh.cand[to] = k; }
                        }
                }
            }
        }
#pragma unroll
        for (int i = 0; i < EACH; i++) x[i] = next[i];
    }

    // ---- threads, warps, CTAs ----
    { uint32_t zero = 0; join_lanes<32>(me, zero); }
    above = __reduce_add_sync(0xffffffffu, above);
    if (lane == 0) { sh.part[warp] = me; sh.above[warp] = above; }
    __syncthreads();
    uint32_t listed = 0;
    if (TOP) {
        if (sh.entering > CAP) {
            __syncthreads();
            if (tid == 0) sh.entering = 0;
            __syncthreads();
            from = 0;
            for (uint32_t at = begin; at < end; at += FOURS * THREADS) {
                load(x, at);
                float big = x[0];
#pragma unroll
                for (int i = 1; i < EACH; i++) big = max_nan(big, x[i]);
                enter(at, big);
            }
            __syncthreads();
        }
        listed = put_in_order(sh, sh.entering, a.top);
    }
    if (warp == 0) {
        me = lane < WARPS ? sh.part[lane] : Triple{-INFINITY, 0, 0};
        above = lane < WARPS ? sh.above[lane] : 0u;
        join_lanes<WARPS>(me, above);
        if (lane == 0) { sh.all = me; sh.all_above = above; sh.listed = listed; }
    }
    cluster_sync();
    if (part == 0) {
        if (TOP && parts > 1) {
            // of every list at least this many reach the least of their places: together no fewer than are wanted
            const uint32_t place = (a.top + parts - 1) / parts - 1, of = min(lane, parts - 1);
            const unsigned long long mark = place < far_u32(there(&sh.listed, of)) ? far_u64(there(&sh.top[place], of)) : 0ull;
            const uint32_t hi = __reduce_min_sync(0xffffffffu, (uint32_t)(mark >> 32));      // by the logits alone
            if (tid == 0) sh.entering = 0;
            __syncthreads();
            for (uint32_t i = tid; i < parts * a.top; i += THREADS) {
                const uint32_t c = i / a.top, j = i % a.top;
                const unsigned long long k = far_u64(there(&sh.top[j], c));
                if (j < far_u32(there(&sh.listed, c)) && (uint32_t)(k >> 32) >= hi) sh.cand[atomicAdd(&sh.entering, 1u)] = k;
            }
        }
        // each warp joins the triples of all CTAs, a lane each
        const uint32_t p = there(&sh.all, min(lane, parts - 1));
        me = Triple{far_f32(p), far_f32(p + 4), far_f32(p + 8)};
        above = far_u32(there(&sh.all_above, min(lane, parts - 1)));
        if (lane >= parts) { me = Triple{-INFINITY, 0, 0}; above = 0; }
        join_lanes<MAX_CLUSTER>(me, above);
        me.m = __shfl_sync(0xffffffffu, me.m, 0); me.s = __shfl_sync(0xffffffffu, me.s, 0);       // one value for all
        const bool none = !(me.m > -INFINITY && me.m < INFINITY);
        const float l = log1pf(me.s), nan = __uint_as_float(0x7fc00000u);
        if (tid == 0) {
            if (a.lp) a.lp[r] = aimed && !none ? (xt - me.m) - l : nan;
            if (a.rank) a.rank[r] = aimed && !none ? above + 1 : 0u;
            if (a.entropy) a.entropy[r] = none ? nan : l - me.w / (1.0f + me.s);
        }
        if (TOP) {
            if (parts > 1) {
                __syncthreads();
                put_in_order(sh, sh.entering, a.top);
                __syncthreads();
            }
            if (tid < a.top) {
                const unsigned long long k = sh.top[tid];
                a.top_ids[r * a.top + tid] = none ? 0xffffffffu : 0xffffffffu - (uint32_t)k;
                a.top_lp[r * a.top + tid] = none ? nan : (key_logit(k) - me.m) - l;
            }
        }
    }
    if (parts > 1) cluster_sync();      // what the first CTA reads stays until it has
}

namespace {
template <bool TOP>
cudaError_t launch(const LogProbArgs& a, uint32_t parts, cudaStream_t st, bool pdl) {
    static bool done[64] = {};
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return err;
    if (dev >= 64 || !done[dev]) {
        err = cudaFuncSetAttribute(log_probs_kernel<TOP>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);      // 16 CTAs
        if (err != cudaSuccess) return err;
        if (dev < 64) done[dev] = true;
    }
    cudaLaunchConfig_t lc = {}; cudaLaunchAttribute at[2];
    lc.gridDim = dim3(a.rows * parts); lc.blockDim = dim3(THREADS); lc.stream = st;
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = parts; at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = at; lc.numAttrs = pdl ? 2 : 1;
    return cudaLaunchKernelEx(&lc, log_probs_kernel<TOP>, a);
}
}  // namespace

cudaError_t launch_log_probs(const LogProbArgs& a, int num_sms, cudaStream_t st, bool pdl) {
    if (!a.rows) return cudaSuccess;
    // The number of parts by what the busiest SM has to do, in logits: a CTA costs about 6000 besides its own, fewer than three do
    // not keep an SM's loads going, and more than are resident at a time (four) cost about 15 %. Measured beside fixed numbers: 64 rows of 128256 11.6 us in 8 parts and 17.3 in 16, 256 of
    // 151643 35.4 in 2 and 37.9 in 4, 300 of 128256 53 in 1 and 38 in 2 or 4.
    uint32_t parts = 1;
    double least = 0;
    for (uint32_t p = 1; p <= MAX_CLUSTER; p *= 2) {
        const double ctas = (double)a.rows * p, per_sm = ctas / num_sms, cost = (ctas <= 4.0 * num_sms ? std::max(3.0, std::ceil(per_sm)) : 1.15 * per_sm) * (6000.0 + (double)a.vocab / p);
        if (p == 1 || cost < least) { least = cost; parts = p; }
    }
    return a.top ? launch<true>(a, parts, st, pdl) : launch<false>(a, parts, st, pdl);
}

}  // namespace alice

using namespace alice;

extern "C" int32_t alice_log_probs(alice_engine* e, const alice_buf* logits, uint32_t rows, uint32_t vocab, size_t stride, const alice_buf* targets, alice_buf* log_probs,
                                   alice_buf* entropy, alice_buf* rank, uint32_t top, alice_buf* top_ids, alice_buf* top_log_probs) {
    const char* who = "alice_log_probs";
    if (!e || !logits) return alice_fail(ALICE_E_INVALID, "%s: null argument", who);
    if (rows > 0x7fffffffu) return alice_fail(ALICE_E_SHAPE, "%s: %u rows", who, rows);
    if (vocab == 0) return alice_fail(ALICE_E_SHAPE, "%s: a vocabulary of none", who);
    if (stride == 0) stride = vocab;
    if (stride < vocab || stride > ((size_t)1 << 40)) return alice_fail(ALICE_E_SHAPE, "%s: rows of %u logits %zu floats apart", who, vocab, stride);
    if (top > LOGP_MAX_TOP || top > vocab) return alice_fail(ALICE_E_SHAPE, "%s: %u alternatives; up to %u, and no more than %u tokens", who, top, LOGP_MAX_TOP, vocab);
    if (!targets && (log_probs || rank)) return alice_fail(ALICE_E_INVALID, "%s: log probabilities and ranks need targets", who);
    if (top && (!top_ids || !top_log_probs)) return alice_fail(ALICE_E_INVALID, "%s: %u alternatives without room for them", who, top);
    if (!rows_fit(logits->len, rows, stride, vocab))
        return alice_fail(ALICE_E_SHAPE, "%s: logits holds %zu words, less than %u rows of %u that are %zu apart", who, logits->len, rows, vocab, stride);
    const size_t read = rows_span(rows, stride, vocab), tops = (size_t)rows * top;
    struct { const char* name; const alice_buf* b; size_t n; bool out; } all[] = {
        {"logits", logits, read, false}, {"targets", targets, rows, false}, {"log_probs", log_probs, rows, true}, {"entropy", entropy, rows, true},
        {"rank", rank, rows, true}, {"top_ids", top ? top_ids : nullptr, tops, true}, {"top_log_probs", top ? top_log_probs : nullptr, tops, true}};
    for (const auto& x : all) {
        if (!x.b) continue;
        if (x.b->e != e) return alice_fail(ALICE_E_INVALID, "%s: %s belongs to another engine", who, x.name);
        if (x.b->len < x.n) return alice_fail(ALICE_E_SHAPE, "%s: %s holds %zu words, %zu are needed", who, x.name, x.b->len, x.n);
        for (const auto& y : all)
            if (x.out && y.b && &y != &x && x.b->p < y.b->p + y.n && y.b->p < x.b->p + x.n)
                return alice_fail(ALICE_E_INVALID, "%s: %s and %s share memory", who, x.name, y.name);
    }
    cudaError_t err = cudaSetDevice(e->device);
    if (err != cudaSuccess) return alice_cuda_fail(err, who);
    auto words = [](alice_buf* b) { return b ? reinterpret_cast<uint32_t*>(b->p) : nullptr; };
    LogProbArgs a{};
    a.x = logits->p; a.ld = stride; a.rows = rows; a.vocab = vocab;
    a.target = targets ? reinterpret_cast<const uint32_t*>(targets->p) : nullptr;
    a.lp = log_probs ? log_probs->p : nullptr; a.entropy = entropy ? entropy->p : nullptr; a.rank = words(rank);
    a.top = top; a.top_ids = top ? words(top_ids) : nullptr; a.top_lp = top ? top_log_probs->p : nullptr;
    err = launch_log_probs(a, e->num_sms, e->stream, e->pdl);
    return err == cudaSuccess ? (int)ALICE_OK : alice_cuda_fail(err, who);
}
