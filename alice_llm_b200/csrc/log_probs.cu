// Log probabilities, entropy, rank and the most probable tokens of rows of logits.
//
// With m the largest logit and s the sum of exp(x - m) over all others but that one:
//   log p(x) = (x - m) - log1p(s),   H = log1p(s) - sum (x - m) exp(x - m) / (1 + s)
// so that what is small beside the largest term is not lost where one token has nearly all the weight.
#include <cmath>

#include "abi_internal.cuh"
#include "common.cuh"
#include "log_probs.cuh"

namespace alice {

namespace {

// Logits in order as whole numbers, the lower index first among equals.
__device__ __forceinline__ unsigned long long logit_key(float x, uint32_t i) {
    const uint32_t u = __float_as_uint(x + 0.0f);      // -0 as 0
    return (unsigned long long)(u & 0x80000000u ? ~u : u | 0x80000000u) << 32 | (0xffffffffu - i);
}

constexpr int LP_THREADS = 256;

template <class T, class F>
__device__ __forceinline__ T over_cta(T v, T* red, F f) {
    __syncthreads();
    red[threadIdx.x] = v;
    __syncthreads();
    for (int o = LP_THREADS / 2; o > 0; o >>= 1) {
        if ((int)threadIdx.x < o) red[threadIdx.x] = f(red[threadIdx.x], red[threadIdx.x + o]);
        __syncthreads();
    }
    return red[0];
}

}  // namespace

// A CTA a row.
__global__ void __launch_bounds__(LP_THREADS) log_probs_kernel(const __grid_constant__ LogProbArgs a) {
    __shared__ unsigned long long keys[LP_THREADS];
    __shared__ float sums[LP_THREADS];
    __shared__ uint32_t counts[LP_THREADS];
    pdl_launch_dependents();
    pdl_wait();
    const size_t r = blockIdx.x;
    const float* x = a.x + r * a.ld;
    auto most = [](unsigned long long p, unsigned long long q) { return p > q ? p : q; };
    auto add = [](float p, float q) { return p + q; };
    auto addu = [](uint32_t p, uint32_t q) { return p + q; };
    unsigned long long best = 0;
    uint32_t odd = 0;
    for (uint32_t i = threadIdx.x; i < a.vocab; i += LP_THREADS) {
        const float v = x[i];
        odd |= !(v < INFINITY);
        best = most(best, logit_key(v, i));
    }
    best = over_cta(best, keys, most);
    odd = over_cta(odd, counts, addu);
    const uint32_t at = 0xffffffffu - (uint32_t)best;
    const float m = x[at];
    const bool none = odd || m == -INFINITY;
    const uint32_t t = a.target ? a.target[r] : 0u;
    const bool valid = a.target && t < a.vocab && !none;
    const float xt = valid ? x[t] : 0.f;
    float s = 0, w = 0;
    uint32_t above = 0;
    for (uint32_t i = threadIdx.x; i < a.vocab; i += LP_THREADS) {
        const float v = x[i], z = fmaxf(v - m, -200.f), e = i == at ? 0.f : expf(z);
        s += e;
        w += e * z;
        above += v > xt;
    }
    s = over_cta(s, sums, add);
    w = over_cta(w, sums, add);
    above = over_cta(above, counts, addu);
    const float l = log1pf(s), nan = __uint_as_float(0x7fc00000u);
    if (threadIdx.x == 0) {
        if (a.lp) a.lp[r] = valid ? (xt - m) - l : nan;
        if (a.rank) a.rank[r] = valid ? above + 1 : 0u;
        if (a.entropy) a.entropy[r] = none ? nan : l - w / (1.f + s);
    }
    unsigned long long below = ~0ull;
    for (uint32_t k = 0; k < a.top; k++) {
        unsigned long long b = 0;
        for (uint32_t i = threadIdx.x; i < a.vocab; i += LP_THREADS) {
            const unsigned long long key = logit_key(x[i], i);
            if (key < below) b = most(b, key);
        }
        below = over_cta(b, keys, most);
        if (threadIdx.x == 0) {
            const uint32_t id = 0xffffffffu - (uint32_t)below;
            a.top_ids[r * a.top + k] = none ? 0xffffffffu : id;
            a.top_lp[r * a.top + k] = none ? nan : (x[id] - m) - l;
        }
    }
}

cudaError_t launch_log_probs(const LogProbArgs& a, int, cudaStream_t st, bool pdl) {
    if (!a.rows) return cudaSuccess;
    cudaLaunchConfig_t lc = {}; cudaLaunchAttribute at[1];
    lc.gridDim = dim3(a.rows); lc.blockDim = dim3(LP_THREADS); lc.stream = st;
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = at; lc.numAttrs = pdl ? 1 : 0;
    return cudaLaunchKernelEx(&lc, log_probs_kernel, a);
}

}  // namespace alice

using namespace alice;

extern "C" int32_t alice_log_probs(alice_engine* e, const alice_buf* logits, uint32_t rows, uint32_t vocab, size_t stride, const alice_buf* targets, alice_buf* log_probs,
                                   alice_buf* entropy, alice_buf* rank, uint32_t top, alice_buf* top_ids, alice_buf* top_log_probs) {
    const char* who = "alice_log_probs";
    if (!e || !logits) return alice_fail(ALICE_E_INVALID, "%s: null argument", who);
    if (vocab == 0) return alice_fail(ALICE_E_SHAPE, "%s: a vocabulary of none", who);
    if (stride == 0) stride = vocab;
    if (stride < vocab || stride > ((size_t)1 << 40)) return alice_fail(ALICE_E_SHAPE, "%s: rows of %u logits %zu floats apart", who, vocab, stride);
    if (top > LOGP_MAX_TOP || top > vocab) return alice_fail(ALICE_E_SHAPE, "%s: %u alternatives; up to %u, and no more than %u tokens", who, top, LOGP_MAX_TOP, vocab);
    if (!targets && (log_probs || rank)) return alice_fail(ALICE_E_INVALID, "%s: log probabilities and ranks need targets", who);
    if (top && (!top_ids || !top_log_probs)) return alice_fail(ALICE_E_INVALID, "%s: %u alternatives without room for them", who, top);
    const size_t read = rows ? (rows - 1) * stride + vocab : 0, tops = (size_t)rows * top;
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
