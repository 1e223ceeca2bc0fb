// lrs_draw.cu — draws from given uniforms with temperature, top-k, top-p and min-p (sm_100a).
//
// The definition (include/llamars_sampler.h) is over the real numbers; the kernel holds every
// weight w = 2^((x - M) log2(e) / T) and every sum in 64 bits, so that a token differs from the
// real-number one only where u falls within about 1e-13 of a step of the distribution function.
#include <cmath>

#include "lrs_ops.cuh"

namespace {

using namespace lrs;

constexpr uint32_t kThreads = 512;
constexpr uint32_t kWarps = kThreads / 32;

// Order-preserving integer of a float (not NaN); -0 and 0 are one value.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

struct Row {
    uint32_t count;
    double mass;
};

__device__ Row block_sum(Row v, Row* part) {
#pragma unroll
    for (int o = 16; o > 0; o /= 2) {
        v.count += __shfl_xor_sync(0xFFFFFFFFu, v.count, o);
        v.mass += __shfl_xor_sync(0xFFFFFFFFu, v.mass, o);
    }
    __syncthreads();
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = v;
    __syncthreads();
    Row t{0, 0.0};
    for (uint32_t w = 0; w < kWarps; ++w) t.count += part[w].count, t.mass += part[w].mass;
    return t;
}

// The sums before this thread's (its own among the total).
__device__ Row block_before(Row v, Row* part, Row* total) {
    Row inc = v;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const uint32_t c = __shfl_up_sync(0xFFFFFFFFu, inc.count, o);
        const double m = __shfl_up_sync(0xFFFFFFFFu, inc.mass, o);
        if ((threadIdx.x & 31) >= o) inc.count += c, inc.mass += m;
    }
    __syncthreads();
    if (threadIdx.x % 32 == 31) part[threadIdx.x / 32] = inc;
    __syncthreads();
    Row t{0, 0.0}, before{0, 0.0};
    for (uint32_t w = 0; w < kWarps; ++w) {
        if (w == threadIdx.x / 32) before = t;
        t.count += part[w].count, t.mass += part[w].mass;
    }
    *total = t;
    const uint32_t c = __shfl_up_sync(0xFFFFFFFFu, inc.count, 1);
    const double m = __shfl_up_sync(0xFFFFFFFFu, inc.mass, 1);
    if (threadIdx.x & 31) before.count += c, before.mass += m;
    return before;
}

// One CTA a row.  The cut in (logit desc, index asc) order is found by bisection over the
// integer order of the logits, a pass over the row a step; the token by one more pass in which
// each thread holds a contiguous piece of the row.
template <typename T>
__global__ void __launch_bounds__(kThreads) draw_kernel(const T* __restrict__ logits, uint32_t n, uint64_t ld,
                                                        const lrs_draw_params* __restrict__ params,
                                                        const float* __restrict__ uniform, uint32_t* __restrict__ tokens,
                                                        float* __restrict__ probs, uint32_t* __restrict__ kept,
                                                        int32_t* __restrict__ status) {
    __shared__ Row part[kWarps];
    __shared__ uint32_t best[kWarps];
    __shared__ float top[kWarps];
    const uint32_t r = blockIdx.x;
    const T* x = logits + r * ld;
    const lrs_draw_params p = params[r];
    const bool greedy = p.temperature <= 0.0f;
    const float u = greedy ? 0.0f : uniform[r];
    auto finish = [&](int32_t st, uint32_t token, float prob, uint32_t count) {
        tokens[r] = token;
        if (probs) probs[r] = prob;
        if (kept) kept[r] = count;
        if (status) status[r] = st;
    };
    if (!isfinite(p.temperature) || (!greedy && (isnan(p.top_p) || !(p.min_p >= 0.0f && p.min_p <= 1.0f) || !(u >= 0.0f && u < 1.0f)))) {
        if (threadIdx.x == 0) finish(LRS_E_INVALID, LRS_TOKEN_NONE, 0.0f, 0);
        return;
    }
    // largest logit, and its lowest index
    float m = -INFINITY;
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) m = max_nan(m, to_float<T>(x[i]));
#pragma unroll
    for (int o = 16; o > 0; o /= 2) m = max_nan(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    if (threadIdx.x % 32 == 0) top[threadIdx.x / 32] = m;
    __syncthreads();
    for (uint32_t w = 0; w < kWarps; ++w) m = max_nan(m, top[w]);
    if (!isfinite(m)) {
        if (threadIdx.x == 0) finish(LRS_E_NAN, LRS_TOKEN_NONE, 0.0f, 0);
        return;
    }
    if (greedy) {
        uint32_t at = n;
        for (uint32_t i = threadIdx.x; i < n && at == n; i += kThreads)
            if (to_float<T>(x[i]) == m) at = i;
        at = __reduce_min_sync(0xFFFFFFFFu, at);
        if (threadIdx.x % 32 == 0) best[threadIdx.x / 32] = at;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (uint32_t w = 0; w < kWarps; ++w) at = min(at, best[w]);
            finish(LRS_OK, at, 1.0f, 1);
        }
        return;
    }
    const double c = 1.4426950408889634 / (double)p.temperature;
    auto weight = [&](float v) { return exp2(((double)v - (double)m) * c); };
    auto at_least = [&](uint32_t key) {  // elements of `key` and above
        Row s{0, 0.0};
        for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
            const float v = to_float<T>(x[i]);
            if (key_of(v) >= key) s.count += 1, s.mass += weight(v);
        }
        return block_sum(s, part);
    };
    const uint32_t lowest = key_of(-INFINITY) + 1;
    const Row all = at_least(lowest);
    const uint32_t k = p.top_k == 0 || p.top_k > n ? n : p.top_k;
    const bool by_mass = p.top_p > 0.0f && p.top_p < 1.0f;
    const double reach = (double)p.top_p * all.mass;
    // the largest key whose elements and those above fill top_k or top_p
    uint32_t lo = lowest, hi = key_of(m) + 1;
    while (hi - lo > 1) {
        const uint32_t mid = lo + (hi - lo) / 2;
        const Row s = at_least(mid);
        if (s.count >= k || (by_mass && s.mass >= reach))
            lo = mid;
        else
            hi = mid;
    }
    uint32_t cut = lo, ties = n;  // elements above the cut, and of its own the first `ties`
    {
        const Row above = at_least(cut + 1);
        const float v = __uint_as_float(cut & 0x80000000u ? cut & 0x7FFFFFFFu : ~cut);
        if (k - above.count < ties) ties = k - above.count;
        if (by_mass) {
            const double w = weight(v);
            double j = floor((reach - above.mass) / w);
            while (above.mass + j * w < reach && j < (double)ties) j += 1.0;
            if (j < 1.0) j = 1.0;
            if (j < (double)ties) ties = (uint32_t)j;
        }
        if (p.min_p > 0.0f) {
            uint32_t a = cut, b = key_of(m);  // smallest key of a weight of min_p, if above the cut
            while (a < b) {
                const uint32_t mid = a + (b - a) / 2;
                if (weight(__uint_as_float(mid & 0x80000000u ? mid & 0x7FFFFFFFu : ~mid)) >= (double)p.min_p)
                    b = mid;
                else
                    a = mid + 1;
            }
            if (a > cut) cut = a, ties = n;
        }
    }
    // the kept elements in vocabulary order: a contiguous piece a thread
    const uint32_t each = (n + kThreads - 1) / kThreads;
    const uint32_t i0 = min(n, threadIdx.x * each), i1 = min(n, i0 + each);
    Row total;
    Row own{0, 0.0};
    for (uint32_t i = i0; i < i1; ++i) own.count += key_of(to_float<T>(x[i])) == cut;
    const uint32_t ties_before = block_before(own, part, &total).count;
    auto piece = [&](auto&& visit) {
        uint32_t seen = ties_before;
        for (uint32_t i = i0; i < i1; ++i) {
            const float v = to_float<T>(x[i]);
            const uint32_t key = key_of(v);
            if (key > cut || (key == cut && seen++ < ties)) {
                if (visit(i, weight(v))) return;
            }
        }
    };
    own = Row{0, 0.0};
    uint32_t last = 0;
    piece([&](uint32_t i, double w) {
        own.count += 1, own.mass += w;
        if (w > 0.0) last = i + 1;
        return false;
    });
    const Row before = block_before(own, part, &total);
    const double target = (double)u * total.mass;
    uint32_t found = n;
    double run = before.mass, wt = 0.0;
    piece([&](uint32_t i, double w) {
        run += w;
        if (run > target) {
            found = i, wt = w;
            return true;
        }
        return false;
    });
    // (sums of two orders differ in their last bits: if none reaches the target, the last weight)
    const uint32_t first = __reduce_min_sync(0xFFFFFFFFu, found);
    const uint32_t end = __reduce_max_sync(0xFFFFFFFFu, last);
    __syncthreads();
    if (threadIdx.x % 32 == 0) best[threadIdx.x / 32] = first, part[threadIdx.x / 32].count = end;
    __syncthreads();
    uint32_t token = n, fall = 0;
    for (uint32_t w = 0; w < kWarps; ++w) token = min(token, best[w]), fall = max(fall, part[w].count);
    if (token == n) {
        token = fall - 1;
        if (threadIdx.x == 0) finish(LRS_OK, token, (float)(weight(to_float<T>(x[token])) / total.mass), total.count);
    } else if (found == token) {
        finish(LRS_OK, token, (float)(wt / total.mass), total.count);
    }
}

template <typename T>
int launch(const void* d_logits, uint32_t rows, uint32_t n, uint64_t ld, const lrs_draw_params* d_params,
           const float* d_uniform, uint32_t* d_tokens, float* d_probs, uint32_t* d_kept, int32_t* d_status,
           cudaStream_t s) {
    draw_kernel<T><<<rows, kThreads, 0, s>>>((const T*)d_logits, n, ld, d_params, d_uniform, d_tokens, d_probs, d_kept, d_status);
    return launched("lrs_draw_device");
}

}  // namespace

extern "C" int lrs_draw_device(const void* d_logits, int dtype, uint32_t rows, uint32_t n, uint64_t ld,
                               const lrs_draw_params* d_params, const float* d_uniform, uint32_t* d_tokens,
                               float* d_probs, uint32_t* d_kept, int32_t* d_status, void* stream) {
    if (rows == 0) return LRS_OK;
    if (dtype != LRS_F32 && dtype != LRS_BF16 && dtype != LRS_F16)
        return lrs_call_error(LRS_E_INVALID, "lrs_draw_device: dtype %d", dtype);
    if (!d_logits || !d_params || !d_uniform || !d_tokens)
        return lrs_call_error(LRS_E_INVALID, "lrs_draw_device: NULL buffer");
    if (n == 0 || n > LRS_DRAW_MAX_VOCAB || rows > LRS_DRAW_MAX_ROWS)
        return lrs_call_error(LRS_E_INVALID, "lrs_draw_device: rows %u / n %u out of range", rows, n);
    if (ld < n && ld != 0) return lrs_call_error(LRS_E_INVALID, "lrs_draw_device: ld < n");
    const uintptr_t size = dtype == LRS_F32 ? 4 : 2;
    if ((uintptr_t)d_logits % size || (uintptr_t)d_params % 4 || (uintptr_t)d_uniform % 4 || (uintptr_t)d_tokens % 4 ||
        (uintptr_t)d_probs % 4 || (uintptr_t)d_kept % 4 || (uintptr_t)d_status % 4)
        return lrs_call_error(LRS_E_INVALID, "lrs_draw_device: a buffer is not aligned to its type");
    auto run = dtype == LRS_F32 ? launch<float> : dtype == LRS_BF16 ? launch<__nv_bfloat16> : launch<__half>;
    return run(d_logits, rows, n, ld, d_params, d_uniform, d_tokens, d_probs, d_kept, d_status, (cudaStream_t)stream);
}
