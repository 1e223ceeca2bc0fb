// lrs_draw.cu — draws from given uniforms with temperature, top-k, top-p and min-p (sm_100a).
//
// The definition (include/llamars_sampler.h) is over the real numbers.  Every weight that decides
// w = 2^((x - M) c), c = log2(e) / T, and every sum of them is held in 64 bits (doubles, or whole
// numbers of 2^-51 of the largest weight), so that a token differs from the real-number one only
// where u falls within about 2e-12 of a step of the distribution function (1e-13 for doubles).
//
// A row is one cluster of CTAs (one CTA for batches, up to 16 for a few rows), each with a slice of
// its tiles of 1024 elements; nothing is kept outside shared memory.
//   1. One pass over the logits: the maximum of every chunk of 128 elements and, where the whole row's
//      mass Z is asked for, the tile's sum of weights, all written to the first CTA (over distributed
//      shared memory).  With filters the sums are 32-bit ones, good to kApprox = 2^-20.
//   2. Few survivors (the first CTA): the k-th largest chunk maximum is a lower bound of the k-th
//      largest logit; maxima whose mass reaches top_p Z bound the nucleus; min-p bounds directly.
//      The chunks that reach the bound are read again, what reaches it goes to a list, the list is
//      sorted and cut; top-p's cut is taken at both ends of Z's error, and Z is summed again in 64
//      bits in the rare case that they differ.  The token comes from the kept list in index order.
//   3. Many survivors (no bound, or a list that overflows; all CTAs): histograms of count and mass
//      over the integer order of the logits narrow the cut to a bracket that fits the list, a last
//      pass sums what lies above it by tile and lists the bracket, and the token is found by tile,
//      then inside one tile.  Without any filter step 1 sums in 64 bits and goes there directly.
// Measured (one B200, passes over changing inputs, f32 rows of 151,936): one row under the default filters 16.4 us, a
// chain of short stages after a pass of 4 us; 1,024 rows under mixed filters 160 to 275 us (199 on average over 24
// inputs; their bytes alone: 95): a row with a large nucleus has one CTA and reads its logits three times, and the batch
// waits for the last such row; 512 rows with nuclei of 12,000 to 119,000 tokens 415 us (48), where step 3 reads the row twice more and the
// 64-bit powers, 17 operations an element of a pipe of half rate, and the levels' additions to shared memory fill the SMs.
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "lrs_ops.cuh"

namespace {

using namespace lrs;
namespace cg = cooperative_groups;

constexpr uint32_t kThreads = 256;
constexpr uint32_t kWarps = kThreads / 32;
constexpr uint32_t kTile = 1024;       // elements of a tile, 32 a lane
constexpr uint32_t kList = 4096;       // candidates that are listed
constexpr uint32_t kChunk = 128;       // elements of a chunk
constexpr uint32_t kPer = kTile / kChunk;
constexpr uint32_t kChunks = 2048;     // chunks that are read again for them
constexpr uint32_t kDirect = kWarps * 12;  // chunks whose candidates are listed with their keys at once
constexpr uint32_t kFew = kThreads;    // candidates that are ranked without a sort
constexpr uint32_t kBins = 4096;
constexpr uint32_t kMaxCluster = 16;
constexpr uint32_t kAll = 0xFFFFFFFFu;
constexpr double kApprox = 0x1p-20;    // of a 32-bit tile sum: ex2.approx 2^-22, its argument 2^-26, six additions deep

// Order-preserving integer of a float (not NaN); -0 and 0 are one value.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}
constexpr uint32_t kLowest = 0x00800000u;  // key of -inf, plus one

__device__ __forceinline__ float warp_max_nan(float v) {
    float r;
    asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}

// 2^y for y <= about 0: the fraction's power by a polynomial (2^f - 1) / f of degree 8 through
// Chebyshev nodes on [-1/2, 1/2], 3.7e-14 off at most and exact at 0; 0 below 2^-1000.  N side by side: a
// chain of 14 operations of the 64-bit pipe is long, and the compiler does not weave unrolled ones.
template <int N>
__device__ __forceinline__ void power2(const double (&y)[N], double (&r)[N]) {
    constexpr double kMagic = 0x1.8p52;
    constexpr double kTerms[9] = {0x1.63d136366db24p-20, 0x1.ffcb9515a8016p-17, 0x1.4308ac85aa947p-13,
                                  0x1.5d87fe86fe88ep-10, 0x1.3b2ab7181b755p-7, 0x1.c6b08d7047e52p-5,
                                  0x1.ebfbdff823cedp-3, 0x1.62e42fefa39efp-1, 1.0};
    double t[N], f[N];
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] = y[i] + kMagic;
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = t[i] - kMagic;
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = y[i] - f[i], r[i] = 0x1.b63880a30e9ffp-24;
#pragma unroll
    for (int k = 0; k < 9; ++k)
#pragma unroll
        for (int i = 0; i < N; ++i) r[i] = fma(r[i], f[i], kTerms[k]);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const bool gone = (uint32_t)__double2hiint(y[i]) > 0xC08F4000u;  // y < -1000, -inf included
        const double p = __hiloint2double(__double2hiint(r[i]) + (__double2loint(t[i]) << 20), __double2loint(r[i]));
        r[i] = gone ? 0.0 : p;
    }
}
__device__ __forceinline__ double power2(double y) {
    const double in[1] = {y};
    double out[1];
    power2(in, out);
    return out[0];
}

// c as a float that 0 can be multiplied by (temperatures below 1e-38 make it larger than any).
__device__ __forceinline__ float finite_float(double c) { return (float)fmin(c, 1e38); }

struct Sum {
    uint32_t n;
    double lo, hi;
};

// Units of a weight of 1 in a bin's mass: the sum of n of them stays below 2^31.
__device__ __forceinline__ uint32_t mass_unit(uint32_t n) { return 1u << (__clz((n - 1) | 1) - 2); }

// How far below the maximum the candidates reach, found from the chunk maxima: the distance in 256ths of the
// maxima's range, and in a second round in 256ths of one of those (a monotone function of x).
struct Bound {
    float top, scale;
    float edge0, edge1;  // inside: distance < edge0 - 1, or within one below edge0 and the rest < edge1
    __device__ __forceinline__ float distance(float x) const { return (0.5f * top - 0.5f * x) * scale; }
    __device__ __forceinline__ bool operator()(float x) const {
        const float f = distance(x);
        return (f < edge0 - 1.0f) | ((f < edge0) & ((f - (edge0 - 1.0f)) * 256.0f < edge1));
    }
};

struct Shared {
    Sum part[kWarps];
    Sum from[kMaxCluster];       // (first CTA: the others' sums)
    float top[kWarps], tops[kMaxCluster];
    uint32_t word[kWarps];
    uint64_t wide[kWarps];
    uint32_t order[4];           // what the first CTA has all do next: operation, upper and lower key, shift
    uint32_t count, chunks;      // entries of the lists
    uint64_t cut;
};

enum { kDone, kLevels, kHistogram, kSumAbove, kGather, kGatherTies, kCandidates };

__device__ __forceinline__ Sum add(const Sum& a, const Sum& b) { return Sum{a.n + b.n, a.lo + b.lo, a.hi + b.hi}; }

__device__ __forceinline__ Sum shift_up(const Sum& v, int o) {
    return Sum{__shfl_up_sync(kAll, v.n, o), __shfl_up_sync(kAll, v.lo, o), __shfl_up_sync(kAll, v.hi, o)};
}

// Sums over the CTA in one order; every thread gets the total, and the sum of the threads before it.
__device__ __noinline__ Sum block_scan(Sum v, Sum* before, Shared& sh) {
    const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    Sum inc = v;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const Sum p = shift_up(inc, o);
        if (lane >= o) inc = add(p, inc);
    }
    __syncthreads();
    if (lane == 31) sh.part[warp] = inc;
    __syncthreads();
    Sum w = lane < kWarps ? sh.part[lane] : Sum{0, 0.0, 0.0};
#pragma unroll
    for (int o = 1; o < (int)kWarps; o *= 2) {
        const Sum p = shift_up(w, o);
        if (lane >= o) w = add(p, w);
    }
    if (before) {
        const Sum in_warp = shift_up(inc, 1);
        const uint32_t last = warp ? warp - 1 : 0;
        const Sum warps{__shfl_sync(kAll, w.n, last), __shfl_sync(kAll, w.lo, last), __shfl_sync(kAll, w.hi, last)};
        Sum r{0, 0.0, 0.0};
        if (warp) r = warps;
        if (lane) r = add(r, in_warp);
        *before = r;
    }
    return Sum{__shfl_sync(kAll, w.n, kWarps - 1), __shfl_sync(kAll, w.lo, kWarps - 1), __shfl_sync(kAll, w.hi, kWarps - 1)};
}

__device__ __noinline__ uint32_t block_min(uint32_t v, Shared& sh) {
    v = __reduce_min_sync(kAll, v);
    __syncthreads();
    if (threadIdx.x % 32 == 0) sh.word[threadIdx.x / 32] = v;
    __syncthreads();
    return __reduce_min_sync(kAll, sh.word[threadIdx.x % kWarps]);
}

__device__ __noinline__ float block_min_float(float v, Shared& sh) {
    const uint32_t key = block_min(key_of(v), sh);
    return value_of(key);
}

// Sums of two words over the threads before each.
__device__ __noinline__ void block_scan_words(uint32_t a, uint32_t b, uint32_t* before_a, uint32_t* before_b, Shared& sh) {
    const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    uint32_t ia = a, ib = b;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const uint32_t qa = __shfl_up_sync(kAll, ia, o), qb = __shfl_up_sync(kAll, ib, o);
        if (lane >= o) ia += qa, ib += qb;
    }
    __syncthreads();
    if (lane == 31) sh.part[warp].n = ia, sh.word[warp] = ib;
    __syncthreads();
    const uint32_t wa = __reduce_add_sync(kAll, lane < warp ? sh.part[lane].n : 0), wb = __reduce_add_sync(kAll, lane < warp ? sh.word[lane] : 0);
    *before_a = wa + ia - a, *before_b = wb + ib - b;
}

// Sum over the threads before each, and of all.
__device__ __noinline__ uint64_t block_scan_long(uint64_t v, uint64_t* before, Shared& sh) {
    const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    uint64_t inc = v;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const uint64_t q = __shfl_up_sync(kAll, inc, o);
        if (lane >= o) inc += q;
    }
    __syncthreads();
    if (lane == 31) sh.wide[warp] = inc;
    __syncthreads();
    uint64_t first = 0, all = 0;
#pragma unroll
    for (uint32_t i = 0; i < kWarps; ++i) {
        if (i == warp) first = all;
        all += sh.wide[i];
    }
    *before = first + inc - v;
    return all;
}

// Bitonic sort of list[0 .. 2^m) (2^m >= count, zeros from count on written here), descending.  Steps
// whose pairs stay within a warp's 64 entries need no barrier of the CTA.
__device__ __noinline__ void sort(uint64_t* list, uint32_t count) {
    uint32_t size = 2;
    while (size < count) size *= 2;
    for (uint32_t i = count + threadIdx.x; i < size; i += kThreads) list[i] = 0;
    __syncthreads();
    for (uint32_t m = 2; m <= size; m *= 2)
        for (uint32_t j = m / 2; j > 0; j /= 2) {
            for (uint32_t t = threadIdx.x; t < size / 2; t += kThreads) {
                const uint32_t i = 2 * t - (t & (j - 1));
                const uint64_t a = list[i], b = list[i + j];
                if ((a < b) == ((i & m) == 0)) list[i] = b, list[i + j] = a;
            }
            if (j > 32 || (j == 1 && m >= 64) || size / 2 > kThreads)
                __syncthreads();
            else
                __syncwarp();
        }
    __syncthreads();
}

// Sums of up to 2^12 whole numbers of up to 2^51 in three words of 17 bits each (32-bit additions to shared
// memory are the ones that the hardware does in place).
__device__ __forceinline__ void add_units(uint32_t* sum, uint64_t units) {
    atomicAdd(sum, (uint32_t)units & 0x1FFFFu);
    atomicAdd(sum + 1, (uint32_t)(units >> 17) & 0x1FFFFu);
    atomicAdd(sum + 2, (uint32_t)(units >> 34));
}
__device__ __forceinline__ uint64_t read_units(const uint32_t* sum) {
    return sum[0] + ((uint64_t)sum[1] << 17) + ((uint64_t)sum[2] << 34);
}

constexpr uint32_t kSlots = 512;  // of the bins below

// Where the kept elements of a list end: `entry` is the last one kept (in descending order), `keep` how
// many are, `sure` whether both ends of Z's error give the same, `filled` whether k or the mass was, or entries had been dropped.
struct Cut {
    uint64_t entry;
    uint32_t keep;
    bool sure, filled;
};

struct Args {
    const void* logits;
    uint64_t ld;
    const lrs_draw_params* params;
    const float* uniform;
    uint32_t* tokens;
    float* probs;
    uint32_t* kept;
    int32_t* status;
    uint32_t n;
    uint32_t twice;  // rows, where the grid goes over them twice (0: once)
    uint32_t most, fill;  // guess_for()
};

// The row as this call sees it: element i at base[i + skew], base on a 16-byte boundary.
template <typename T>
struct RowView {
    static constexpr uint32_t kVec = 16 / sizeof(T), kLoad = 32 * kVec, kLoads = kTile / kLoad;  // of a warp
    const T* base;
    uint32_t skew, end;  // elements are base[skew .. end)

    // -inf, kVec (or two words of it: half) times
    static __device__ __forceinline__ uint32_t nothing() {
        return sizeof(T) == 4 ? 0xFF800000u : std::is_same<T, __half>::value ? 0xFC00FC00u : 0xFF80FF80u;
    }
    __device__ __forceinline__ bool holds(uint32_t j, uint32_t count) const { return (j >= skew) & (j + count <= end); }
    // count elements from position j some of which are outside the row: -inf there
    template <uint32_t COUNT>
    __device__ __forceinline__ void piece(uint32_t j, float* v) const {
        T x[COUNT];
#pragma unroll
        for (uint32_t i = 0; i < COUNT; ++i) x[i] = base[min(max(j + i, skew), end - 1)];  // (in flight together)
#pragma unroll
        for (uint32_t i = 0; i < COUNT; ++i) v[i] = holds(j + i, 1) ? to_float<T>(x[i]) : -INFINITY;
    }
    // four elements from position j (a multiple of four), all within the row
    __device__ __forceinline__ void whole_quad(uint32_t j, float (&v)[4]) const {
        if constexpr (sizeof(T) == 4) {
            unpack(__ldg(reinterpret_cast<const uint4*>(base + j)), v, base);
        } else {
            const uint2 q = __ldg(reinterpret_cast<const uint2*>(base + j));
            float x[8];
            unpack(make_uint4(q.x, q.y, 0, 0), x, base);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = x[i];
        }
    }
    __device__ __forceinline__ void quad(uint32_t j, float (&v)[4]) const {
        if (holds(j, 4))
            whole_quad(j, v);
        else
            piece<4>(j, v);
    }
    // A lane's 32 elements of a tile, -inf outside the row.  The loads go out together, those of the row's
    // ends too: taken one after the other there, a tile took 8 us and not 1.
    __device__ __forceinline__ void tile(uint32_t t, float (&v)[32]) const {
        const uint32_t j = t * kTile + threadIdx.x % 32 * kVec;
        uint4 r[kLoads];
        const bool inner = holds(t * kTile, kTile);
        if (inner) {
#pragma unroll
            for (uint32_t c = 0; c < kLoads; ++c) r[c] = __ldg(reinterpret_cast<const uint4*>(base + j + c * kLoad));
        } else {
#pragma unroll
            for (uint32_t c = 0; c < kLoads; ++c) {
                r[c] = make_uint4(nothing(), nothing(), nothing(), nothing());
                if (holds(j + c * kLoad, kVec)) r[c] = __ldg(reinterpret_cast<const uint4*>(base + j + c * kLoad));
            }
        }
#pragma unroll
        for (uint32_t c = 0; c < kLoads; ++c) {
            float x[kVec];
            unpack(r[c], x, base);
#pragma unroll
            for (uint32_t i = 0; i < kVec; ++i) v[c * kVec + i] = x[i];
        }
        if (inner) return;
#pragma unroll
        for (uint32_t c = 0; c < kLoads; ++c) {  // (a vector at either end)
            const uint32_t at = j + c * kLoad;
            if (!holds(at, kVec) && at < end && at + kVec > skew) piece<kVec>(at, v + c * kVec);
        }
    }
    // the maxima of the tile's chunks: lane i < kPer gets chunk i's; a NaN stays
    __device__ __forceinline__ float chunk_max(const float (&v)[32], float* all) const {
        const uint32_t lane = threadIdx.x % 32;
        float mine = 0.0f, top = -INFINITY;
#pragma unroll
        for (uint32_t c = 0; c < kLoads; ++c) {
            float m = v[c * kVec];
#pragma unroll
            for (uint32_t e = 1; e < kVec; ++e) m = max_nan(m, v[c * kVec + e]);
            constexpr uint32_t kIn = kLoad / kChunk;  // chunks of a load: 1, or one a half-warp
#pragma unroll
            for (uint32_t h = 0; h < kIn; ++h) {
                const float w = warp_max_nan(kIn == 1 || lane / 16 == h ? m : -INFINITY);
                if (lane == c * kIn + h) mine = w;
                top = max_nan(top, w);
            }
        }
        *all = top;
        return mine;
    }
};

constexpr int kWeave = 4;

// Weights relative to a maximum.
struct Weigh {
    double max, c;
    __device__ __forceinline__ double operator()(float x) const { return power2(((double)x - max) * c); }
    template <int N>
    __device__ __forceinline__ void many(const float* x, double (&w)[N]) const {
        double y[N];
#pragma unroll
        for (int i = 0; i < N; ++i) y[i] = ((double)x[i] - max) * c;
        power2(y, w);
    }
    // the sum of a lane's 32
    __device__ __forceinline__ double sum(const float (&v)[32]) const {
        double s[kWeave] = {};
#pragma unroll
        for (int i = 0; i < 32; i += kWeave) {
            double w[kWeave];
            many(v + i, w);
#pragma unroll
            for (int j = 0; j < kWeave; ++j) s[j] += w[j];
        }
#pragma unroll
        for (int j = 1; j < kWeave; ++j) s[0] += s[j];
        return s[0];
    }
};

// 32-bit tile sums: 2^(x c) = 2^f 2^k, k the nearest integer to x c and f the rest, exact to 2^-26
// through two fused steps; sums are relative to 2^K, K the tile maximum's k.
struct Rough {
    float hi, lo;
    static constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23
    __device__ __forceinline__ bool fits(float top) const { return hi > 1e-30f && fabsf(top) * hi <= 0x1p20f; }
    __device__ __forceinline__ float unit(float top) const { return fmaf(top, hi, kMagic) - kMagic; }
    __device__ __forceinline__ float sum(const float (&v)[32], float top) const {
        const float least = top - 120.0f / hi;
        const int32_t k0 = __float_as_int(fmaf(top, hi, kMagic));
        float s[8];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const float x = fmaxf(v[i], least);
            const float t = fmaf(x, hi, kMagic);
            const float f = fmaf(x, lo, fmaf(x, hi, -(t - kMagic)));
            float e;
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(f));
            const float w = __int_as_float(__float_as_int(e) + ((__float_as_int(t) - k0) << 23));
            s[i / 4] = i % 4 == 0 ? w : s[i / 4] + w;
        }
#pragma unroll
        for (int o = 4; o > 0; o /= 2)
#pragma unroll
            for (int i = 0; i < o; ++i) s[i] += s[i + o];
        return s[0];
    }
};

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o > 0; o /= 2) v += __shfl_xor_sync(kAll, v, o);
    return v;
}

// Room on the first CTA's list for the elements of the lanes' bit masks: one addition to its count a warp.
__device__ __forceinline__ uint32_t reserve(uint32_t* count, uint32_t mask) {
    const uint32_t lane = threadIdx.x % 32, mine = __popc(mask);
    uint32_t inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const uint32_t q = __shfl_up_sync(kAll, inc, o);
        if (lane >= o) inc += q;
    }
    uint32_t at = 0;
    if (lane == 31) at = atomicAdd(count, inc);
    return __shfl_sync(kAll, at, 31) + inc - mine;
}
// Appends them.
template <int N, typename At>
__device__ __forceinline__ void append(uint64_t* list, uint32_t* count, const float (&v)[N], uint32_t mask, At index) {
    if (!__any_sync(kAll, mask != 0)) return;
    uint32_t at = reserve(count, mask);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const bool hit = mask >> i & 1;
        if (hit & (at < kList)) list[at] = (uint64_t)key_of(v[i]) << 32 | ~index(i);
        at += hit;
    }
}
// Appends their indices alone, for fill_list(): a turn a hit, where append() has one an element (with that one
// the gathering pass of a row of 151,936 took 106 us and not 86, the list of 3,700 candidates 62 and not 36).
template <typename At>
__device__ __forceinline__ void append_indices(uint64_t* list, uint32_t* count, uint32_t mask, At index) {
    if (!__any_sync(kAll, mask != 0)) return;
    uint32_t at = reserve(count, mask);
    for (; mask; mask &= mask - 1, ++at)
        if (at < kList) list[at] = ~index(__ffs(mask) - 1);
}

// The first CTA's copy of shared memory (its own for itself: the cluster's window is slower).
template <typename P>
__device__ __forceinline__ P* of_first(P* p) {
    cg::cluster_group cluster = cg::this_cluster();
    return cluster.block_rank() ? cluster.map_shared_rank(p, 0) : p;
}

// What every CTA does with its slice of the row when the first CTA says so (sh.order).
template <typename T>
struct Slice {
    RowView<T> row;
    uint32_t t0, t1, n;  // tiles of the slice, elements of the row
    double c;
    uint8_t* dynamic;    // (as the kernel lays it out)
    double* first_sum;
    float* first_max;
    __device__ __forceinline__ uint32_t index(uint32_t t, int i) const {  // of element i of a lane's 32
        return t * kTile + i / RowView<T>::kVec * RowView<T>::kLoad + threadIdx.x % 32 * RowView<T>::kVec + i % RowView<T>::kVec - row.skew;
    }
};

// The keys of a list of indices (the first CTA).
template <typename T>
__device__ __noinline__ void fill_list(const RowView<T>& row, uint64_t* list, uint32_t count) {
    constexpr uint32_t kAhead = 8;
    for (uint32_t i = threadIdx.x; i < count; i += kThreads * kAhead) {
        uint32_t low[kAhead];
        T x[kAhead];
#pragma unroll
        for (uint32_t a = 0; a < kAhead; ++a) low[a] = (uint32_t)list[i + a * kThreads < count ? i + a * kThreads : i];
#pragma unroll
        for (uint32_t a = 0; a < kAhead; ++a) x[a] = row.base[~low[a] + row.skew];
#pragma unroll
        for (uint32_t a = 0; a < kAhead; ++a)
            if (i + a * kThreads < count) list[i + a * kThreads] = (uint64_t)key_of(to_float<T>(x[a])) << 32 | low[a];
    }
    __syncthreads();
}

// Candidates: the elements from `least` up, to the first CTA's list, from the chunks that it has listed
// (shared out over all warps).  Four chunks at a time, the next four on their way meanwhile.  Of more than
// kDirect chunks the indices alone are listed.
template <typename T>
__device__ __noinline__ void list_candidates(const Slice<T>& z, Shared& sh) {
    constexpr uint32_t kGroup = 4;
    cg::cluster_group cluster = cg::this_cluster();
    uint64_t* first_list = of_first(reinterpret_cast<uint64_t*>(z.dynamic));
    const uint32_t* again = reinterpret_cast<const uint32_t*>(first_list + kList);
    uint32_t* first_count = of_first(&sh.count);
    const float least = value_of(sh.order[2]);
    const uint32_t reaching = sh.order[1], lane = threadIdx.x % 32;
    const uint32_t step = sh.order[3] * kWarps * kGroup;  // (CTAs that share the chunks)
    uint32_t i = (cluster.block_rank() * kWarps + threadIdx.x / 32) * kGroup;
    auto load = [&](uint32_t first, uint32_t (&from)[kGroup], float (&v)[4 * kGroup]) {
        bool whole_chunks = true;
#pragma unroll
        for (uint32_t q = 0; q < kGroup; ++q) {
            from[q] = again[min(first + q, reaching - 1)] * kChunk;  // (past the end: the last again, not listed)
            whole_chunks &= z.row.holds(from[q], kChunk);
            from[q] += lane * 4;
        }
        if (whole_chunks) {
#pragma unroll
            for (uint32_t q = 0; q < kGroup; ++q) z.row.whole_quad(from[q], *reinterpret_cast<float(*)[4]>(&v[4 * q]));
        } else {
#pragma unroll
            for (uint32_t q = 0; q < kGroup; ++q) z.row.template piece<4>(from[q], v + 4 * q);
        }
    };
    if (i >= reaching) return;
    uint32_t from[kGroup];
    float v[4 * kGroup];
    load(i, from, v);
    while (true) {
        const uint32_t next = i + step;
        uint32_t from_next[kGroup];
        float v_next[4 * kGroup];
        if (next < reaching) load(next, from_next, v_next);
        uint32_t mask = 0;
#pragma unroll
        for (uint32_t q = 0; q < 4 * kGroup; ++q) mask |= (v[q] >= least) & (i + q / 4 < reaching) ? 1u << q : 0u;
        if (reaching > kDirect)
            append_indices(first_list, first_count, mask, [&](int q) { return again[i + q / 4] * kChunk + lane * 4 + q % 4 - z.row.skew; });
        else
            append(first_list, first_count, v, mask, [&](int q) { return from[q / 4] + q % 4 - z.row.skew; });
        if (next >= reaching) return;
        i = next;
#pragma unroll
        for (uint32_t q = 0; q < kGroup; ++q) from[q] = from_next[q];
#pragma unroll
        for (uint32_t q = 0; q < 4 * kGroup; ++q) v[q] = v_next[q];
    }
}

// Where bin b is kept: a word is left free after every kEachBin bins, a thread's share of them, so that
// threads that read their shares meet all banks.
constexpr uint32_t kEachBin = kBins / kThreads;
constexpr uint32_t kBinWords = kBins + kThreads;
__device__ __forceinline__ uint32_t bin_place(uint32_t b) { return b + b / kEachBin; }

// Each CTA adds up a part of the bins over all CTAs, into the first one's.
__device__ __forceinline__ void merge_bins(uint32_t* bins, uint32_t words) {
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t ctas = cluster.num_blocks(), rank = cluster.block_rank();
    if (ctas == 1) return;
    cluster.sync();
    const uint32_t each = words / ctas;  // (a whole number for 1, 2, 4, 8, 16)
    for (uint32_t i = rank * each + threadIdx.x; i < (rank + 1) * each; i += kThreads) {
        uint32_t sum = 0;
#pragma unroll 4
        for (uint32_t q = 0; q < ctas; ++q) sum += cluster.map_shared_rank(bins, q)[i];
        cluster.map_shared_rank(bins, 0)[i] = sum;
    }
}

// A logit's level: its distance from the maximum in steps of 1 / steps, to the nearest; monotone.
__device__ __forceinline__ uint32_t level_of(float x, float max, float steps) {
    return __float_as_uint(fmaf(max - x, steps, 8388608.0f)) - 0x4B000000u;
}

// Counts of the levels 0 .. kBins - 1, to the first CTA's bins (clear before).  A level's weights differ by
// so little that its mass is its count times the middle one: one addition an element.
template <typename T>
__device__ __noinline__ void count_levels(const Slice<T>& z, float max, Shared& sh) {
    const float steps = __uint_as_float(sh.order[1]);
    uint32_t* bin_n = reinterpret_cast<uint32_t*>(z.dynamic);
    if (cg::this_cluster().block_rank()) {
        for (uint32_t i = threadIdx.x; i < kBinWords; i += kThreads) bin_n[i] = 0;
        __syncthreads();
    }
    const uint32_t spare = threadIdx.x % 32 * (kEachBin + 1) + kEachBin;
    for (uint32_t t = z.t0 + threadIdx.x / 32; t < z.t1; t += kWarps) {
        float v[32];
        z.row.tile(t, v);
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const uint32_t b = level_of(v[i], max, steps);
            atomicAdd(&bin_n[b < kBins ? bin_place(b) : spare], 1u);
        }
    }
    merge_bins(bin_n, kBinWords);
}

// A power of two above a bin's weights: 2^edge, by at most a factor of four (round to nearest by addition).
__device__ __forceinline__ float bin_edge(uint32_t key, float max, float c) {
    return (fmaxf((value_of(key) - max) * c, -1000.0f) + 12582912.0f) - 12582911.0f;
}

// Counts and masses of the keys of [lo, hi) in bins of 2^shift keys, the highest first, to the first CTA's
// bins (clear before); returns the count and mass (64 bits) of the keys above.
template <typename T>
__device__ __noinline__ Sum histogram(const Slice<T>& z, float max, Shared& sh) {
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t hi = sh.order[1], lo = sh.order[2], shift = sh.order[3];
    uint32_t* bin_n = reinterpret_cast<uint32_t*>(z.dynamic);
    uint32_t* bin_w = bin_n + kBinWords;
    const uint32_t rank = cluster.block_rank();
    if (rank) {
        for (uint32_t i = threadIdx.x; i < 2 * kBinWords; i += kThreads) bin_n[i] = 0;
        __syncthreads();
    }
    const Weigh weigh{(double)max, z.c};
    const float cf = finite_float(z.c), scale = (float)min(mass_unit(z.n), 1u << 22);
    Sum s{0, 0.0, 0.0};
    for (uint32_t t = z.t0 + threadIdx.x / 32; t < z.t1; t += kWarps) {
        float v[32];
        z.row.tile(t, v);
        uint32_t above = 0;
        // (without a branch, so that the chains overlap: what is outside goes to words that no bin uses)
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const uint32_t key = key_of(v[i]);
            const uint32_t b = (hi - 1 - key) >> shift;
            float e;
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"((v[i] - max) * cf - bin_edge(hi - 1 - (b << shift), max, cf)));
            const uint32_t w = __float_as_uint(fmaf(fminf(e, 1.0f), scale, 8388608.0f)) - 0x4B000000u;  // (below 2^23)
            above |= key >= hi ? 1u << i : 0u;
            const uint32_t place = (key >= lo) & (key < hi) ? bin_place(b) : threadIdx.x % 32 * (kEachBin + 1) + kEachBin;
            atomicAdd(&bin_n[place], 1u);
            atomicAdd(&bin_w[place], w);
        }
        if (__any_sync(kAll, above != 0)) {
            s.n += __popc(above);
#pragma unroll
            for (int i = 0; i < 32; i += kWeave) {
                double w[kWeave];
                weigh.many(v + i, w);
#pragma unroll
                for (int j = 0; j < kWeave; ++j) s.lo += above >> (i + j) & 1 ? w[j] : 0.0;
            }
        }
    }
    merge_bins(bin_n, 2 * kBinWords);
    return s;
}

// Sums in 64 bits of the keys from hi up and of all, by tile as well (kSumAbove: not by tile); the keys
// of [lo, hi) go to the first CTA's list, or (kGatherTies) are counted by tile.
template <typename T>
__device__ __noinline__ Sum gather(const Slice<T>& z, float max, Shared& sh) {
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t op = sh.order[0], lane = threadIdx.x % 32;
    const float from = value_of(sh.order[1]), least = value_of(sh.order[2]);
    uint64_t* first_list = of_first(reinterpret_cast<uint64_t*>(z.dynamic));
    uint32_t* first_count = of_first(&sh.count);
    const Weigh weigh{(double)max, z.c};
    Sum s{0, 0.0, 0.0};
    for (uint32_t t = z.t0 + threadIdx.x / 32; t < z.t1; t += kWarps) {
        float v[32];
        z.row.tile(t, v);
        double above = 0.0, all = 0.0;
        uint32_t mask = 0;
#pragma unroll
        for (int i = 0; i < 32; i += kWeave) {
            double w[kWeave];
            weigh.many(v + i, w);
#pragma unroll
            for (int j = 0; j < kWeave; ++j) {
                const float x = v[i + j];
                all += w[j];
                above += x >= from ? w[j] : 0.0;
                s.n += x >= from;
                mask |= (x >= least) & (x < from) ? 1u << (i + j) : 0u;
            }
        }
        s.lo += above, s.hi += all;
        if (op == kSumAbove) continue;
        above = warp_sum(above);
        if (lane == 0) z.first_sum[t] = above;
        if (op == kGatherTies) {
            const uint32_t ties = __reduce_add_sync(kAll, __popc(mask));
            if (lane == 0) reinterpret_cast<uint32_t*>(z.first_max)[t] = ties;
        } else {
            append_indices(first_list, first_count, mask, [&](int i) { return z.index(t, i); });
        }
    }
    return s;
}

template <typename T>
__device__ void perform(const Slice<T>& z, float max, Shared& sh) {
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t op = sh.order[0];
    Sum s{0, 0.0, 0.0};
    if (op == kCandidates)
        list_candidates(z, sh);
    else if (op == kLevels)
        count_levels(z, max, sh);
    else
        s = op == kHistogram ? histogram(z, max, sh) : gather(z, max, sh);
    s = block_scan(s, nullptr, sh);
    if (threadIdx.x == 0) *cluster.map_shared_rank(&sh.from[cluster.block_rank()], 0) = s;
    if (cluster.num_blocks() > 1)
        cluster.sync();
    else
        __syncthreads();
}

// A weight in whole numbers of 2^-51: their sums do not depend on an order.
__device__ __forceinline__ uint64_t units(const Weigh& weigh, uint64_t entry) {
    return __double2ull_rn(weigh(value_of((uint32_t)(entry >> 32))) * 0x1p51);
}
// The same where the token is found: one unit at least for every weight that is not 0, so that u = 0 draws the
// first kept element however light it is (a list's 2^12 entries shift the steps by 2^-39 at most).
__device__ __forceinline__ uint64_t drawn_units(double w) {
    const uint64_t whole = __double2ull_rn(w * 0x1p51);
    return whole == 0 && w > 0.0 ? 1 : whole;
}
// What of `reach` is left above `base`, in the same units.
__device__ __forceinline__ uint64_t units_left(double reach, double base) {
    return __double2ull_ru(fmin(fmax(reach - base, 0.0) * 0x1p51, 0x1p63));
}

// The cut of a list (zeros: dropped entries) below base_n kept elements of mass base: the entries are dealt
// into slots by their value between the list's ends, the slots' counts and masses summed from the top,
// and the entries of the slot that fills k or `reach` compared with one another.  A slot that too many
// share (long runs of nearly equal values) has the list sorted instead.
__device__ __noinline__ Cut find_cut(uint64_t* list, uint32_t* slots, uint32_t* members, uint32_t count, uint32_t base_n,
                                     double base, uint32_t k, bool by_mass, double reach_lo, double reach_hi,
                                     const Weigh weigh, Shared& sh) {
    uint32_t least = kAll, most = 0, mine = 0;
    for (uint32_t i = threadIdx.x; i < count; i += kThreads) {
        const uint32_t key = (uint32_t)(list[i] >> 32);
        if (key) least = min(least, key), most = max(most, key), ++mine;
    }
    const uint32_t least_key = block_min(least, sh);
    const float low = value_of(least_key), top = value_of(~block_min(~most, sh));
    const uint32_t real = block_scan(Sum{mine, 0.0, 0.0}, nullptr, sh).n;
    if (real == 0) return Cut{~0ull, 0, true, false};
    auto all = [&] {  // every entry is kept: the lowest of them
        uint32_t last = kAll;
        for (uint32_t i = threadIdx.x; i < count; i += kThreads)
            if ((uint32_t)(list[i] >> 32) == least_key) last = min(last, (uint32_t)list[i]);
        return Cut{(uint64_t)least_key << 32 | block_min(last, sh), real, true, k - base_n <= real || real < count};
    };
    if (!by_mass && k - base_n >= real) return all();
    const float scale = low < top ? fminf((float)kSlots * 0.999f / (0.5f * top - 0.5f * low), 0x1p100f) : 1.0f;
    auto slot_of = [&](uint64_t entry) {
        return min((uint32_t)((0.5f * top - 0.5f * value_of((uint32_t)(entry >> 32))) * scale), kSlots - 1);
    };
    const uint64_t goal_lo = by_mass ? units_left(reach_lo, base) : ~0ull, goal_hi = by_mass ? units_left(reach_hi, base) : ~0ull;
    const uint32_t goal_n = k - base_n;
    uint32_t* slot_n = slots;            // counts, and masses of three words
    uint32_t* slot_w = slots + kSlots;
    for (uint32_t i = threadIdx.x; i < 4 * kSlots; i += kThreads) slots[i] = 0;
    if (threadIdx.x == 0) sh.chunks = 0;
    __syncthreads();
#pragma unroll 4
    for (uint32_t i = threadIdx.x; i < count; i += kThreads) {
        const uint64_t e = list[i];
        if (!e) continue;
        const uint32_t at = slot_of(e);
        atomicAdd(&slot_n[at], 1u);
        if (by_mass) add_units(slot_w + 3 * at, units(weigh, e));
    }
    __syncthreads();
    const uint32_t one = 2 * threadIdx.x, two = one + 1;
    uint32_t before_n, unused;
    uint64_t before = 0, w1 = 0, w2 = 0;
    block_scan_words(slot_n[one] + slot_n[two], 0, &before_n, &unused, sh);
    if (by_mass) {
        w1 = read_units(slot_w + 3 * one), w2 = read_units(slot_w + 3 * two);
        block_scan_long(w1 + w2, &before, sh);
    }
    const uint32_t n1 = before_n + slot_n[one], n2 = n1 + slot_n[two];
    auto hit = [&](uint64_t goal) {
        const uint32_t at = n1 >= goal_n || before + w1 >= goal ? one : n2 >= goal_n || before + w1 + w2 >= goal ? two : kAll;
        return block_min(at, sh);
    };
    const uint32_t at = hit(goal_lo), at_hi = by_mass ? hit(goal_hi) : at;
    if (at != at_hi) return Cut{0, 0, false, false};
    if (at == kAll) return all();
    if (at == one || at == two) sh.count = at == one ? before_n : n1, sh.cut = at == one ? before : before + w1;
    for (uint32_t i = threadIdx.x; i < count; i += kThreads) {
        if (!list[i] || slot_of(list[i]) != at) continue;
        const uint32_t m = atomicAdd(&sh.chunks, 1u);
        if (m < kThreads) members[m] = i;
    }
    __syncthreads();
    const uint32_t in = sh.chunks, above_n = sh.count;
    const uint64_t above = sh.cut;
    __syncthreads();
    if (in <= kThreads) {
        uint64_t* mass = reinterpret_cast<uint64_t*>(slots);  // (the slots have served)
        const uint64_t e = threadIdx.x < in ? list[members[threadIdx.x]] : 0;
        if (by_mass && e) mass[threadIdx.x] = units(weigh, e);
        __syncthreads();
        uint32_t rank = above_n;
        uint64_t over = above;
        if (e)
            for (uint32_t j = 0; j < in; ++j) {
                const bool more = list[members[j]] > e;
                rank += more;
                if (by_mass) over += more ? mass[j] : 0;
            }
        const bool keep = e && rank < goal_n && over < goal_lo, keep_hi = e && rank < goal_n && over < goal_hi;
        if (__syncthreads_or(keep != keep_hi)) return Cut{0, 0, false, false};
        const uint32_t kept = __syncthreads_count(keep);
        // (none: there was nothing left to fill; else the last one kept is one of the slot that fills it)
        if (kept == 0) return Cut{~0ull, 0, true, true};
        if (keep && rank + 1 == above_n + kept) sh.cut = e;
        __syncthreads();
        return Cut{sh.cut, above_n + kept, true, true};
    }
    sort(list, count);
    const uint32_t per = (real + kThreads - 1) / kThreads;
    const uint32_t i0 = min(real, threadIdx.x * per), i1 = min(real, i0 + per);
    uint64_t sum = 0, run;
    if (by_mass)
        for (uint32_t i = i0; i < i1; ++i) sum += units(weigh, list[i]);
    block_scan_long(sum, &run, sh);
    uint32_t a = 0, b = 0;
    for (uint32_t i = i0; i < i1; ++i) {
        a += i < goal_n && run < goal_lo, b += i < goal_n && run < goal_hi;
        if (by_mass) run += units(weigh, list[i]);
    }
    const uint32_t keep = block_scan(Sum{a, 0.0, 0.0}, nullptr, sh).n, keep_hi = block_scan(Sum{b, 0.0, 0.0}, nullptr, sh).n;
    return Cut{keep ? list[keep - 1] : ~0ull, keep, keep == keep_hi, true};
}

// Three CTAs an SM leave 80 registers, of which some 800 bytes a thread are spilled over the kernel; two leave 128 and 48
// bytes.  Three and two, us (one B200, f32 rows of 151,936, graph replays over three inputs): 1,024 mixed 162 and 184, 1,024
// default filters 160 and 182, 1,024 unfiltered 236 and 270, 512 large nuclei 416 and 384, 256 x 109,051 bf16 min-p 50.6 and 48.6,
// one row 15.4 and 14.6: batches of several waves need the third, the others lose 4 to 8 % by it.
template <typename T>
__global__ void __launch_bounds__(kThreads, 3) draw_kernel(const Args g) {
    extern __shared__ __align__(16) uint8_t dynamic[];
    __shared__ Shared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t ctas = cluster.num_blocks(), rank = cluster.block_rank();
    const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    uint32_t r = blockIdx.x / ctas;
    const bool again_over = g.twice && r >= g.twice;
    if (again_over) r -= g.twice;
    auto all_sync = [&] {
        if (ctas > 1)
            cluster.sync();
        else
            __syncthreads();
    };

    const lrs_draw_params p = g.params[r];
    const bool greedy = p.temperature <= 0.0f;
    // (rows that may keep tens of thousands of tokens take several passes: they go first)
    const bool deep = !greedy && (p.top_k == 0 || p.top_k > kList) && !(p.min_p > 0.0f);
    if (g.twice && deep == again_over) return;
    const float u = greedy ? 0.0f : g.uniform[r];
    auto finish = [&](int32_t st, uint32_t token, double prob, uint32_t count) {
        g.tokens[r] = token;
        if (g.probs) g.probs[r] = (float)prob;
        if (g.kept) g.kept[r] = count;
        if (g.status) g.status[r] = st;
    };
    if (!isfinite(p.temperature) || (!greedy && (isnan(p.top_p) || !(p.min_p >= 0.0f && p.min_p <= 1.0f) || !(u >= 0.0f && u < 1.0f)))) {
        if (rank == 0 && threadIdx.x == 0) finish(LRS_E_INVALID, LRS_TOKEN_NONE, 0.0, 0);
        return;  // (every CTA of the cluster)
    }
    const uint32_t n = g.n;
    RowView<T> row;
    {
        const T* x = reinterpret_cast<const T*>(g.logits) + r * g.ld;
        row.skew = (uint32_t)((uintptr_t)x % 16 / sizeof(T));
        row.base = x - row.skew;
        row.end = n + row.skew;
    }
    const uint32_t tiles = (row.end + kTile - 1) / kTile, chunks = tiles * kPer;
    const uint32_t each = (tiles + ctas - 1) / ctas, t0 = min(tiles, rank * each), t1 = min(tiles, t0 + each);

    uint64_t* list = reinterpret_cast<uint64_t*>(dynamic);                 // kList entries, or
    uint32_t* bin_n = reinterpret_cast<uint32_t*>(dynamic);                // kBinWords counts and
    uint32_t* bin_w = bin_n + kBinWords;                                   // masses (into `again`)
    static_assert(2 * kBinWords * 4 <= kList * 8 + kChunks * 4, "the bins fit the lists' memory");
    uint32_t* again = reinterpret_cast<uint32_t*>(list + kList);           // kChunks chunk numbers
    uint32_t* slots = again + kChunks;                                     // 4 kSlots words
    double* tile_sum = reinterpret_cast<double*>(slots + 4 * kSlots);      // a tile's
    float* chunk_max = reinterpret_cast<float*>(tile_sum + (tiles + 1) / 2 * 2);
    double* first_sum = of_first(tile_sum);
    float* first_max = of_first(chunk_max);

    const uint32_t k = p.top_k == 0 || p.top_k > n ? n : p.top_k;
    const bool by_mass = p.top_p > 0.0f && p.top_p < 1.0f;
    const bool whole = !greedy && k == n && !by_mass && !(p.min_p > 0.0f);  // no filter
    const double c = 1.4426950408889634 / (double)p.temperature;
    const Rough rough{(float)c, (float)(c - (double)(float)c)};

    // ---- 1. one pass: chunk maxima and tile sums ----
    if (ctas > 1) cluster.sync();  // (the first CTA is there to be written to)
    float top = -INFINITY;
    uint32_t open = 0;             // elements above -inf
    for (uint32_t t = t0 + warp; t < t1; t += kWarps) {
        float v[32];
        row.tile(t, v);
        float tile_top;
        const float mine = row.chunk_max(v, &tile_top);
        if (lane < kPer) first_max[t * kPer + lane] = mine;
        top = max_nan(top, tile_top);
        if (!(by_mass || whole) || greedy) continue;
        double s = 0.0;
        if (isfinite(tile_top)) {
            if (!whole && rough.fits(tile_top)) {
                s = warp_sum((double)rough.sum(v, tile_top));
            } else {
                s = warp_sum(Weigh{(double)tile_top, c}.sum(v));
            }
            if (whole) {
#pragma unroll
                for (int i = 0; i < 32; ++i) open += v[i] > -INFINITY;
            }
        }
        if (lane == 0) first_sum[t] = s;
    }
    if (lane == 0) sh.top[warp] = top;
    __syncthreads();
    for (uint32_t w = 0; w < kWarps; ++w) top = max_nan(top, sh.top[w]);
    if (whole) open = block_scan(Sum{open, 0.0, 0.0}, nullptr, sh).n;
    if (ctas > 1) {
        if (threadIdx.x == 0) {
            *cluster.map_shared_rank(&sh.tops[rank], 0) = top;
            cluster.map_shared_rank(&sh.from[rank], 0)->n = open;
        }
        cluster.sync();
        if (rank == 0) {
            open = 0;
            for (uint32_t q = 0; q < ctas; ++q) top = max_nan(top, sh.tops[q]), open += sh.from[q].n;
        }
    }

    // The first CTA leads; `order` tells the others what to do.
    auto command = [&](uint32_t op, uint32_t hi, uint32_t lo, uint32_t shift) {
        __syncthreads();
        if (threadIdx.x < ctas) {
            uint32_t* o = cluster.map_shared_rank(sh.order, threadIdx.x);
            o[0] = op, o[1] = hi, o[2] = lo, o[3] = shift;
        }
        all_sync();
    };
    const Slice<T> slice{row, t0, t1, n, c, dynamic, first_sum, first_max};
    if (rank != 0) {
        while (true) {
            all_sync();
            if (sh.order[0] == kDone) return;
            perform(slice, *cluster.map_shared_rank(&sh.tops[0], 0), sh);
        }
    }

    // ---- the first CTA from here on ----
    auto total = [&] {  // what a perform() summed, over the CTAs
        Sum s = sh.from[0];
        for (uint32_t q = 1; q < ctas; ++q) s = add(s, sh.from[q]);
        return s;
    };
    auto leave = [&] {
        if (ctas > 1) command(kDone, 0, 0, 0);
    };
    if (!isfinite(top)) {
        if (threadIdx.x == 0) finish(LRS_E_NAN, LRS_TOKEN_NONE, 0.0, 0);
        return leave();
    }
    if (ctas > 1 && threadIdx.x == 0) sh.tops[0] = top;
    if (greedy) {
        uint32_t at = chunks;
        for (uint32_t i = threadIdx.x; i < chunks && at == chunks; i += kThreads)
            if (chunk_max[i] == top) at = i;
        at = block_min(at, sh);
        if (warp == 0) {
            float v[4];
            const uint32_t j = at * kChunk + lane * 4;
            row.quad(j, v);
            uint32_t index = kAll;
#pragma unroll
            for (int e = 3; e >= 0; --e)
                if (v[e] == top) index = j + e - row.skew;
            index = __reduce_min_sync(kAll, index);
            if (lane == 0) finish(LRS_OK, index, 1.0, 1);
        }
        return leave();
    }
    const Weigh weigh{(double)top, c};
    // a tile's sum relative to the row's maximum
    auto tile_mass = [&](uint32_t t) {
        float m = -INFINITY;
#pragma unroll
        for (uint32_t i = 0; i < kPer; ++i) m = fmaxf(m, chunk_max[t * kPer + i]);
        if (m == -INFINITY) return 0.0;
        if (!whole && rough.fits(m)) return tile_sum[t] * power2((double)rough.unit(m) - (double)top * c);
        return tile_sum[t] * weigh(m);
    };
    double z = 0.0;  // the whole row's mass
    if (by_mass) {
        Sum s{0, 0.0, 0.0};
        for (uint32_t t = threadIdx.x; t < tiles; t += kThreads) s.lo += tile_mass(t);
        z = block_scan(s, nullptr, sh).lo;
    }
    const double top_p = (double)p.top_p;
    double reach_lo = by_mass ? top_p * z * (1.0 - kApprox) : INFINITY, reach_hi = by_mass ? top_p * z * (1.0 + kApprox) : INFINITY;

    auto units_of = [&](uint64_t entry) { return drawn_units(weigh(value_of((uint32_t)(entry >> 32)))); };
    // Entries lighter than min_p leave the list.
    auto drop_light = [&](uint32_t count) {
        if (p.min_p > 0.0f) {
#pragma unroll 4
            for (uint32_t i = threadIdx.x; i < count; i += kThreads)
                if (!(weigh(value_of((uint32_t)(list[i] >> 32))) >= (double)p.min_p)) list[i] = 0;
        }
        __syncthreads();
    };

    if (!whole) {
        // ---- 2. few survivors ----
        float least = value_of(kLowest);  // nothing lighter than min_p is kept
        if (p.min_p > 0.0f) {
            const double below = log2((double)p.min_p) / c;
            least = fmaxf(least, __double2float_rd((double)top + below - (fabs((double)top) - below) * 1e-12));
        }
        // How far below the maximum the list has to go: the chunk maxima alone fill top_k or top_p there.
        uint32_t* few_n = reinterpret_cast<uint32_t*>(dynamic);  // counts of a bin
        uint32_t* few_w = few_n + kThreads;                      // masses, in units that never round up
        float low = top;
        for (uint32_t i = threadIdx.x; i < chunks; i += kThreads)
            if (chunk_max[i] >= least) low = fminf(low, chunk_max[i]);
        low = block_min_float(low, sh);
        const uint32_t unit = min(mass_unit(chunks), 1u << 24);
        const uint64_t mass_goal = by_mass ? __double2ull_ru(fmin(reach_hi * unit, 0x1p40)) : ~0ull;
        Bound bound{top, low < top ? fminf(255.9f / (0.5f * top - 0.5f * low), 0x1p100f) : 1.0f, 0.0f, 1e30f};  // (halves: no overflow)
        // Where they do not fill either, the bound goes down to where the list is as good as full, g.most maxima
        // (guess_for()), whatever the values if they come in no order: a list that may do, and shows it if it
        // does.  It is tried where k is at most what it then holds, g.fill, or the mass above the bound seems to
        // be enough: if a share 1 - i / N of the chunks has nothing above x, -ln(1 - i / N) elements a chunk lie
        // there, so that the i-th largest maximum stands for N / (N - i) elements.  "Enough" begins at 0.96 of the
        // goal: at 0.90 rows whose nucleus is a little too long listed in vain (1,024 x 151,936, sigma 3, top_p 0.9 in
        // 842 us, 670 at 0.98), at 0.98 rows that would do went on (Zipf-like, top_p 0.85-0.95: 272 us, 199 at 0.94).
        const uint32_t most = g.most;
        bool guess = false, bounded = true;
        uint32_t reaching = 0;
        for (int round = 0; round < 2; ++round) {
            few_n[threadIdx.x] = 0, few_w[threadIdx.x] = 0;
            __syncthreads();
            uint32_t above = 0, above_w = 0;
            for (uint32_t i = threadIdx.x; i < chunks; i += kThreads) {
                const float m = chunk_max[i];
                if (!(m >= least)) continue;
                float f = bound.distance(m);
                const uint32_t w = by_mass ? __double2uint_rd(weigh(m) * unit) : 0u;
                if (round == 1) {
                    if (f < bound.edge0 - 1.0f) above += 1, above_w += w;
                    if (!(f >= bound.edge0 - 1.0f && f < bound.edge0)) continue;
                    f = (f - (bound.edge0 - 1.0f)) * 256.0f;
                }
                const uint32_t b = min((uint32_t)f, kThreads - 1);
                atomicAdd(&few_n[b], 1u);
                if (by_mass) atomicAdd(&few_w[b], w);
            }
            if (above) atomicAdd(&few_n[0], above), atomicAdd(&few_w[0], above_w);  // (counted with the first bin)
            __syncthreads();
            const uint32_t bin = threadIdx.x;
            uint32_t before_n, before_w;
            block_scan_words(few_n[bin], few_w[bin], &before_n, &before_w, sh);
            const uint32_t upto = before_n + few_n[bin];
            const bool fills = guess ? upto >= most : upto >= k || (uint64_t)before_w + few_w[bin] >= mass_goal;
            uint32_t at = block_min(fills ? bin : kAll, sh);
            if (at == kAll && n > kList && (by_mass || k < n)) {
                const uint32_t edge = block_min(upto >= most ? bin : kAll, sh);
                Sum held{0, 0.0, 0.0};
                if (bin <= edge) held.lo = few_w[bin] * ((double)chunks / (chunks - min(before_n + few_n[bin] / 2, chunks - 1)));
                guess = k <= g.fill || (by_mass && block_scan(held, nullptr, sh).lo >= 0.96 * (double)mass_goal);
                if (guess) at = edge;
            }
            if (at == kAll) {  // not even all of them: every element from `least` up
                bounded = false;
                break;
            }
            if (bin == at) sh.count = upto;
            __syncthreads();
            reaching = sh.count;
            if (round == 0)
                bound.edge0 = (float)(at + 1);
            else
                bound.edge1 = (float)(at + 1);
            if (reaching <= (guess ? most + 16 : k < chunks ? k + 32 : 64)) break;
            __syncthreads();
        }
        bounded = bounded && !bound(least);  // (or what passes `least` is all there is)
        guess = guess && bounded;
        float from = least;                                    // candidates: from here up
        if (bounded) {
            from = top;
            for (uint32_t i = threadIdx.x; i < chunks; i += kThreads)
                if (chunk_max[i] >= least && bound(chunk_max[i])) from = fminf(from, chunk_max[i]);
            from = block_min_float(from, sh);
        }
        __syncthreads();
        if (threadIdx.x == 0) sh.count = 0, sh.chunks = 0;
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < chunks; i += kThreads) {
            if (!(chunk_max[i] >= from)) continue;
            const uint32_t at = atomicAdd(&sh.chunks, 1u);
            if (at < kChunks) again[at] = i;
        }
        __syncthreads();
        // (without a bound the list would be the row)
        reaching = bounded || p.min_p > 0.0f || n <= kList ? sh.chunks : kAll;
        if (reaching <= kChunks) {
            if (ctas > 1 && reaching > kDirect) {  // many chunks: all CTAs
                command(kCandidates, reaching, key_of(from), ctas);
                perform(slice, top, sh);
            } else {
                if (threadIdx.x == 0) sh.order[1] = reaching, sh.order[2] = key_of(from), sh.order[3] = 1;
                __syncthreads();
                list_candidates(slice, sh);
            }
            __syncthreads();
            const uint32_t count = sh.count;
            if (reaching > kDirect && count <= kList) fill_list(row, list, count);
            auto row_mass = [&] {  // Z again, in 64 bits
                Sum s{0, 0.0, 0.0};
                for (uint32_t t = warp; t < tiles; t += kWarps) {
                    float v[32];
                    row.tile(t, v);
                    s.lo += weigh.sum(v);
                }
                return block_scan(s, nullptr, sh).lo;
            };
            if (count <= kFew && !guess) {
                // Every candidate's rank and the mass before it by comparison with all, the comparisons of
                // one shared by `lanes` neighbours; masses are whole numbers of 2^-51, so that their sums do
                // not depend on the list's order.
                uint32_t lanes = 1;
                while (lanes < 32 && count * lanes * 2 <= kThreads) lanes *= 2;
                const uint32_t me = threadIdx.x / lanes, part = threadIdx.x % lanes;
                const bool real = me < count;
                uint64_t* mass = list + kFew;   // of every candidate
                const uint64_t entry = real ? list[me] : 0;
                const double w = real ? weigh(value_of((uint32_t)(entry >> 32))) : 0.0;
                const uint64_t units = __double2ull_rn(w * 0x1p51);
                if (real && part == 0) mass[me] = units;
                __syncthreads();
                uint32_t rank = 0;
                uint64_t before = 0;
                if (real)
                    for (uint32_t j = part; j < count; j += lanes) {
                        const bool over = list[j] > entry;
                        rank += over;
                        before += over ? mass[j] : 0;
                    }
                for (uint32_t o = 1; o < lanes; o *= 2) {
                    rank += __shfl_xor_sync(kAll, rank, o);
                    before += __shfl_xor_sync(kAll, before, o);
                }
                auto kept_to = [&](double reach) {
                    return real && rank < k && w >= (double)p.min_p && (!by_mass || before < __double2ull_ru(fmin(reach * 0x1p51, 0x1p63)));
                };
                bool keep = kept_to(reach_lo);
                if (__syncthreads_or(keep != kept_to(reach_hi))) {  // Z's error decides
                    z = row_mass();
                    keep = kept_to(top_p * z);
                }
                const uint64_t drawn = keep ? drawn_units(w) : 0;
                if (real && part == 0) mass[me] = drawn;
                const uint32_t kept = __syncthreads_count(keep && part == 0);
                const uint32_t index = ~(uint32_t)entry;
                uint64_t upto = 0, total = 0;
                if (real)
                    for (uint32_t j = part; j < count; j += lanes) {
                        const uint64_t m = mass[j];
                        total += m;
                        upto += ~(uint32_t)list[j] <= index ? m : 0;
                    }
                for (uint32_t o = 1; o < lanes; o *= 2) {
                    total += __shfl_xor_sync(kAll, total, o);
                    upto += __shfl_xor_sync(kAll, upto, o);
                }
                const bool passes = drawn && (double)upto > (double)u * (double)total;
                uint32_t token = block_min(passes ? index : kAll, sh);
                if (token == kAll) token = ~block_min(drawn ? ~index : kAll, sh);  // (u's product rounded up: the last)
                if (real && part == 0 && index == token) finish(LRS_OK, token, w * 0x1p51 / (double)total, kept);
                return leave();
            }
            while (count <= kList) {
                Cut kept{1, 0, true, true};
                const bool light = p.min_p > 0.0f && !by_mass && k >= n;  // min_p alone: tested below
                if (!light) {
                    drop_light(count);
                    kept = find_cut(list, slots, again, count, 0, 0.0, k, by_mass, reach_lo, reach_hi, weigh, sh);
                    if (!kept.sure) {  // Z's error decides
                        z = row_mass();
                        kept = find_cut(list, slots, again, count, 0, 0.0, k, by_mass, top_p * z, top_p * z, weigh, sh);
                    }
                }
                if (guess && !kept.filled) break;
                const uint64_t cut = kept.entry;
                // The token: masses (whole numbers of 2^-51: their sums know no order) by ranges of indices,
                // the range that the target falls in again by parts where it is crowded, then its entries.
                uint32_t* range = slots;  // three words each
                uint32_t first = 0, width = (n + kSlots - 1) / kSlots;  // indices from `first`, `width` a range
                uint64_t below = 0, total = 0;
                double target = 0.0;
                uint32_t mine = 0;
                for (int round = 0; round < 2; ++round) {
                    __syncthreads();
                    for (uint32_t i = threadIdx.x; i < 3 * kSlots; i += kThreads) range[i] = 0;
                    if (threadIdx.x == 0) sh.count = 0;
                    __syncthreads();
#pragma unroll 4
                    for (uint32_t i = threadIdx.x; i < count; i += kThreads) {
                        const uint64_t e = list[i];
                        const uint32_t slot = (~(uint32_t)e - first) / width;  // (before `first`: out of range too)
                        if (e < cut || slot >= kSlots) continue;
                        const double w = weigh(value_of((uint32_t)(e >> 32)));
                        if (light && !(w >= (double)p.min_p)) {
                            list[i] = 0;
                            continue;
                        }
                        mine += round == 0;
                        add_units(range + 3 * slot, drawn_units(w));
                    }
                    __syncthreads();
                    const uint64_t a = read_units(range + 6 * threadIdx.x), b = read_units(range + 6 * threadIdx.x + 3);
                    uint64_t before;
                    const uint64_t all = block_scan_long(a + b, &before, sh);
                    before += below;
                    if (round == 0) total = all, target = (double)u * (double)total;
                    uint32_t hit = (double)(before + a) > target ? 2 * threadIdx.x : (double)(before + a + b) > target ? 2 * threadIdx.x + 1 : kAll;
                    hit = block_min(hit, sh);
                    if (hit == kAll) hit = ~block_min(b ? ~(2 * threadIdx.x + 1) : a ? ~(2 * threadIdx.x) : kAll, sh);  // (u's product rounded up: the last)
                    if (threadIdx.x == hit / 2) sh.cut = hit % 2 ? before + a : before;
                    __syncthreads();
                    below = sh.cut;
                    first += hit * width;
                    for (uint32_t i = threadIdx.x; i < count; i += kThreads) {
                        const uint64_t e = list[i];
                        if (e < cut || ~(uint32_t)e - first >= width) continue;
                        const uint32_t at = atomicAdd(&sh.count, 1u);
                        if (at < kThreads) again[at] = i;
                    }
                    __syncthreads();
                    if (sh.count <= kThreads) break;
                    width = (width + kSlots - 1) / kSlots;  // (at most 2^22 / 512 / 512 = 16 indices then)
                }
                const uint32_t members = sh.count;
                if (light) kept.keep = block_scan(Sum{mine, 0.0, 0.0}, nullptr, sh).n;
                const uint64_t entry = threadIdx.x < members ? list[again[threadIdx.x]] : 0;
                const uint32_t index = ~(uint32_t)entry;
                uint64_t upto = below;
                if (entry)
                    for (uint32_t j = 0; j < members; ++j) {
                        const uint64_t e = list[again[j]];
                        if (~(uint32_t)e <= index) upto += units_of(e);
                    }
                const bool weighs = entry && units_of(entry);
                uint32_t token = block_min(weighs && (double)upto > target ? index : kAll, sh);
                if (token == kAll) token = ~block_min(weighs ? ~index : kAll, sh);
                if (entry && index == token)
                    finish(LRS_OK, token, weigh(value_of((uint32_t)(entry >> 32))) * 0x1p51 / (double)total, kept.keep);
                return leave();
            }
        }
    }

    // ---- 3. many survivors ----
    uint64_t cut = (uint64_t)kLowest << 32;  // kept: key << 32 | ~index from here up
    uint32_t tie_key = 0, tie_keep = 0;      // or, of this key, the first tie_keep in index order
    uint32_t kept = open;
    if (whole) {
        for (uint32_t t = threadIdx.x; t < tiles; t += kThreads) tile_sum[t] = tile_mass(t);
    } else {
        uint32_t lo = kLowest, hi = key_of(top) + 1;
        if (p.min_p > 0.0f) {
            const double below = log2((double)p.min_p) / c;
            lo = max(lo, key_of(__double2float_rd((double)top + below - (fabs((double)top) - below) * 1e-12)));
        }
        const double rest = (1.0 - top_p) * z;  // what may be left out
        bool all_below = true;                  // min_p leaves out no more than that
        if (by_mass) {  // what is lighter than rest / n is left out even if every element is; 2^-10 of that for the levels
            const double below = log2(rest * (1.0 - 2.0 * kApprox) * 0x1p-10 / n) / c;
            const uint32_t lightest = key_of(__double2float_rd((double)top + below - (fabs((double)top) + fabs(below)) * 1e-12));
            all_below = lightest >= lo;
            lo = max(lo, lightest);
        }
        if (hi <= lo) lo = hi - 1;
        uint32_t inside = kAll;  // elements of [lo, hi)
        Sum base{0, 0.0, 0.0};   // count and mass from hi up
        // levels of the weights' logarithm down to the lightest that may be kept, where those are fine ones
        const float steps = fminf((float)(kBins - 8) / (top - value_of(lo)), 0x1p100f);
        const float octaves = finite_float(c) / steps;  // of a level
        if (by_mass && hi - lo > 1 && octaves <= 1.0f) {
            __syncthreads();
            for (uint32_t i = threadIdx.x; i < kBinWords; i += kThreads) bin_n[i] = 0;
            command(kLevels, __float_as_uint(steps), 0, 0);
            perform(slice, top, sh);
            // (a level's weights lie within half of one of its middle, but for the roundings of 32 bits)
            const double off = (double)exp2f(0.501f * octaves) - 1.0 + 0x1p-14;
            Sum s{0, 0.0, 0.0}, before;
            auto add_level = [&](uint32_t b, Sum* run) {
                const uint32_t m = bin_n[bin_place(b)];
                run->n += m, run->lo += (double)m * (double)exp2f(-(float)b * octaves);
            };
            for (uint32_t i = 0; i < kEachBin; ++i) add_level(threadIdx.x * kEachBin + i, &s);
            const double counted = block_scan(s, &before, sh).lo;
            uint32_t a = kBins - 1, z1 = kBins - 1;
            for (uint32_t i = 0; i < kEachBin; ++i) {
                const uint32_t b = threadIdx.x * kEachBin + i;
                add_level(b, &before);
                // (the mass above against top_p Z, and the mass below against the rest of Z: the one is good near
                // the top, the other where top_p leaves little; what lies under the levels is 2^-10 of the rest, but
                // for what min_p leaves out there: then only the first says that the cut is reached)
                const double under = counted - before.lo;
                const bool may = before.lo * (1.0 + off) >= reach_lo && under * (1.0 - off) <= rest * (1.0 + kApprox);
                const bool does = before.lo * (1.0 - off) >= reach_hi ||
                                  (all_below && under * (1.0 + off) + rest * 0x1p-9 <= rest * (1.0 - kApprox));
                if ((before.n >= k || may) && b < a) a = b;
                if ((before.n >= k || does) && b < z1) z1 = b;
            }
            const uint32_t last = min(level_of(value_of(lo), top, steps), kBins - 1);  // (nothing fills: the lightest)
            a = min(block_min(a, sh), last), z1 = min(block_min(z1, sh), last);
            s = Sum{0, 0.0, 0.0};
            for (uint32_t b = a + threadIdx.x; b <= z1; b += kThreads) s.n += bin_n[bin_place(b)];
            inside = block_scan(s, nullptr, sh).n;
            // the levels' ends as keys: the lowest key of a level up to `level`
            auto lowest = [&](uint32_t level) {
                uint32_t under = kLowest - 1, from = hi - 1;  // (the maximum is of level 0)
                while (from - under > 1) {
                    const uint32_t mid = under + (from - under) / 2;
                    if (level_of(value_of(mid), top, steps) <= level)
                        from = mid;
                    else
                        under = mid;
                }
                return from;
            };
            lo = max(lo, lowest(z1));
            if (a > 0) hi = lowest(a - 1);
            if (hi <= lo) lo = hi - 1;
        }
        for (int round = 0; round < 3 && inside > kList && (hi - lo > 1 || round == 0); ++round) {
            const uint32_t range = hi - lo;
            const uint32_t bits = 32 - __clz(range - 1 | 1);
            const uint32_t shift = bits > 12 ? bits - 12 : 0;
            __syncthreads();
            for (uint32_t i = threadIdx.x; i < 2 * kBinWords; i += kThreads) bin_n[i] = 0;
            command(kHistogram, hi, lo, shift);
            perform(slice, top, sh);
            base = total();
            // where the cut may lie: counts are exact, masses within their rounding (half a unit an
            // element, and the 32-bit power), Z within its own; masses here in 2^-40
            const float cf = finite_float(c);
            const int unit = 31 - __clz(min(mass_unit(n), 1u << 22));  // a bin's masses are in 2^(edge - unit)
            auto fixed = [](double mass) { return __double2ull_rd(fmin(fmax(mass, 0.0) * 0x1p40, 0x1p63)); };
            auto bin = [&](uint32_t b, uint64_t* lo_mass, uint64_t* hi_mass) {
                const uint32_t w = bin_w[bin_place(b)], m = bin_n[bin_place(b)];
                if (m == 0 || !by_mass) return m;
                const int up = (int)bin_edge(hi - 1 - (b << shift), top, cf), left = up + 40 - unit;
                if (left <= -32) {  // (weighs nothing)
                    *hi_mass += 1;
                    return m;
                }
                auto at = [&](uint64_t v) { return left >= 0 ? v << left : v >> -left; };
                const uint64_t l = at(w > m ? w - m : 0), h = at((uint64_t)w + m) + 1;
                const uint64_t err = (uint64_t)(3 - up);  // in 2^-20 of the mass
                *lo_mass += l - min(l, (l >> 20) * err + err), *hi_mass += h + (h >> 20) * err + err;
                return m;
            };
            uint32_t own_n = 0, before_n, unused;
            uint64_t own_lo = 0, own_hi = 0, run_lo, run_hi;
            for (uint32_t i = 0; i < kEachBin; ++i) own_n += bin(threadIdx.x * kEachBin + i, &own_lo, &own_hi);
            block_scan_words(own_n, 0, &before_n, &unused, sh);
            block_scan_long(own_lo, &run_lo, sh);
            block_scan_long(own_hi, &run_hi, sh);
            run_lo += fixed(base.lo), run_hi += fixed(base.lo) + 1;
            const uint64_t goal_lo = by_mass ? fixed(reach_lo) : ~0ull, goal_hi = by_mass ? fixed(reach_hi) + 1 : ~0ull;
            uint32_t run_n = base.n + before_n, a = kBins - 1, z1 = kBins - 1;
            for (uint32_t i = 0; i < kEachBin; ++i) {
                const uint32_t b = threadIdx.x * kEachBin + i;
                run_n += bin(b, &run_lo, &run_hi);
                if ((run_n >= k || run_hi >= goal_lo) && b < a) a = b;
                if ((run_n >= k || run_lo >= goal_hi) && b < z1) z1 = b;
            }
            a = block_min(a, sh), z1 = block_min(z1, sh);
            const uint32_t last = (range - 1) >> shift;
            a = min(a, last), z1 = min(z1, last);
            Sum in{0, 0.0, 0.0};
            for (uint32_t b = a + threadIdx.x; b <= z1; b += kThreads) in.n += bin_n[bin_place(b)];
            inside = block_scan(in, nullptr, sh).n;
            const uint32_t from = hi;
            hi = from - (a << shift);
            lo = max(lo, from - min(from, (z1 + 1) << shift));
        }
        // (histograms that do not settle, as with a mass far below their unit: halves, summed exactly)
        if (inside > kList && hi - lo > 1) {
            command(kSumAbove, hi, hi, 0);
            perform(slice, top, sh);
            uint32_t above = total().n;
            const double reach = by_mass ? top_p * total().hi : INFINITY;
            command(kSumAbove, lo, lo, 0);
            perform(slice, top, sh);
            uint32_t upto = total().n;
            while (upto - above > kList && hi - lo > 1) {
                const uint32_t mid = lo + (hi - lo) / 2;
                command(kSumAbove, mid, mid, 0);
                perform(slice, top, sh);
                const Sum s = total();
                if (s.n >= k || s.lo >= reach)
                    lo = mid, upto = s.n;
                else
                    hi = mid, above = s.n;
            }
            inside = upto - above;
        }
        const bool ties = inside > kList;  // (of one key)
        __syncthreads();
        if (threadIdx.x == 0) sh.count = 0;
        command(ties ? kGatherTies : kGather, hi, lo, 0);
        perform(slice, top, sh);
        const Sum above = total();
        const double reach = by_mass ? top_p * above.hi : INFINITY;  // (Z in 64 bits)
        if (ties) {
            tie_key = lo;
            const double w = weigh(value_of(lo));
            double j = (double)min(inside, k - above.n);
            if (by_mass) {
                double q = w > 0.0 ? fmax(1.0, floor((reach - above.lo) / w)) : j;
                while (q < j && above.lo + q * w < reach) q += 1.0;
                j = fmin(j, q);
            }
            if (w < (double)p.min_p) j = 0.0;
            tie_keep = (uint32_t)j;
            kept = above.n + tie_keep;
            cut = (uint64_t)hi << 32;
            // each tile's share, in index order
            uint32_t* tile_ties = reinterpret_cast<uint32_t*>(chunk_max);
            const uint32_t per = (tiles + kThreads - 1) / kThreads;
            const uint32_t i0 = min(tiles, threadIdx.x * per), i1 = min(tiles, i0 + per);
            Sum s{0, 0.0, 0.0}, before;
            for (uint32_t t = i0; t < i1; ++t) s.n += tile_ties[t];
            block_scan(s, &before, sh);
            uint32_t seen = before.n;
            for (uint32_t t = i0; t < i1; ++t) {
                const uint32_t has = tile_ties[t], keep = seen >= tie_keep ? 0 : min(has, tie_keep - seen);
                seen += has;
                tile_ties[t] = keep;
                tile_sum[t] += keep * w;
            }
        } else {
            const uint32_t count = min(sh.count, kList);
            fill_list(row, list, count);
            drop_light(count);
            const Cut end = find_cut(list, slots, again, count, above.n, above.lo, k, by_mass, reach, reach, weigh, sh);
            cut = end.keep ? end.entry : (uint64_t)hi << 32;
            kept = above.n + end.keep;
            // (the chunks' maxima have served: each tile's share of the list, in units whose sums know no order)
            uint32_t* share = reinterpret_cast<uint32_t*>(chunk_max);
            for (uint32_t t = threadIdx.x; t < 3 * tiles; t += kThreads) share[t] = 0;
            __syncthreads();
#pragma unroll 4
            for (uint32_t i = threadIdx.x; i < count; i += kThreads)
                if (list[i] >= cut) add_units(share + 3 * ((~(uint32_t)list[i] + row.skew) / kTile), units_of(list[i]));
            __syncthreads();
            for (uint32_t t = threadIdx.x; t < tiles; t += kThreads) tile_sum[t] += (double)read_units(share + 3 * t) * 0x1p-51;
        }
    }
    leave();
    __syncthreads();
    // the tile that holds the token, and what lies before it
    const uint32_t per = (tiles + kThreads - 1) / kThreads;
    const uint32_t i0 = min(tiles, threadIdx.x * per), i1 = min(tiles, i0 + per);
    Sum s{0, 0.0, 0.0}, before;
    for (uint32_t t = i0; t < i1; ++t) s.lo += tile_sum[t];
    const double mass = block_scan(s, &before, sh).lo, target = (double)u * mass;
    uint32_t at = kAll, heavy = 0;
    double run = before.lo, base = 0.0;
    // (a tile without weight holds nothing that is kept: a thread's `run` may exceed its neighbour's last one by a bit,
    // since the sums before it are added in another order, and a target on that step would stop at such a tile)
    for (uint32_t t = i0; t < i1; ++t) {
        if (tile_sum[t] > 0.0) {
            heavy = t + 1;
            if (at == kAll && run + tile_sum[t] > target) at = t, base = run;
        }
        run += tile_sum[t];
    }
    uint32_t tile = block_min(at, sh);
    if (tile == kAll) {  // (two orders of a sum: the last tile with weight)
        tile = ~block_min(~heavy, sh) - 1;
        base = INFINITY;
        if (threadIdx.x == 0) sh.part[0].lo = base;
    } else if (at == tile) {
        sh.part[0].lo = base;
    }
    __syncthreads();
    // inside the tile, four elements a thread
    base = sh.part[0].lo;
    const uint32_t quota = tie_keep ? reinterpret_cast<uint32_t*>(chunk_max)[tile] : 0;
    const uint32_t j = tile * kTile + threadIdx.x * 4;
    float v[4];
    row.quad(j, v);
    uint32_t tied = 0;
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) tied += tie_keep && key_of(v[e]) == tie_key;
    uint32_t seen = 0;
    if (tie_keep) {
        uint32_t unused;
        block_scan_words(tied, 0, &seen, &unused, sh);
    }
    double w[4];
    s = Sum{0, 0.0, 0.0};
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) {
        const uint32_t key = key_of(v[e]);
        bool in = key >= kLowest && ((uint64_t)key << 32 | ~(j + e - row.skew)) >= cut;
        if (tie_keep && key == tie_key) in = seen++ < quota;
        w[e] = in ? weigh(v[e]) : 0.0;
        s.lo += w[e];
    }
    block_scan(s, &before, sh);
    double here = base + before.lo, w_first = 0.0, w_last = 0.0;
    uint32_t first = kAll, end = 0;
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) {
        here += w[e];
        if (w[e] > 0.0) {
            if (first == kAll && here > target && base < INFINITY) first = j + e - row.skew, w_first = w[e];
            end = j + e - row.skew + 1, w_last = w[e];
        }
    }
    uint32_t token = block_min(first, sh);
    if (token == kAll) {  // (two orders of a sum: the last one with weight)
        token = ~block_min(~end, sh) - 1;
        if (end == token + 1) finish(LRS_OK, token, w_last / mass, kept);
    } else if (first == token) {
        finish(LRS_OK, token, w_first / mass, kept);
    }
}

constexpr int kMaxDevices = 64;

template <typename T>
size_t shared_bytes(uint32_t n) {
    const uint32_t tiles = (n + 15 + kTile - 1) / kTile;
    return kList * 8 + kChunks * 4 + kSlots * 16 + (tiles + 1) / 2 * 2 * 8 + (size_t)tiles * kPer * 4;
}

// The guessed list of rows of n elements: `most`, how many of the N chunk maxima it takes in, and `fill`, how many
// elements it then holds more often than not.  With j maxima left below the bound, the elements above it are N times the
// (j + 1)-th smallest of N exponential variables turned over: N ln((N + 1/2) / (j + 1/2)) of them, N / sqrt(j + 0.6) their
// standard deviation.  j is the least that leaves two and a half of those to the list's end (a row in a hundred overflows at
// most), has its chunks listed, and is 4.5 % of N: longer lists make short rows' nuclei slower (256 x 32,003, 532 kept: 34.9 us,
// 40.3 with every maximum taken in) and hardly fill more of them.  So 1,133 of 1,187 maxima at n = 151,936, 3,660 +- 160
// elements; 238 of 250 at 32,003, 750 +- 70; 1,422 of 1,562 at 200,000, 3,760 +- 130.  Sizes that the list does not hold
// are not guessed (48 x 32,003 fp16, k = 1,000: 43.0 us, 52.3 guessed in vain; 256 x 65,000, k = 2,500: 106 and 126), and long rows'
// lists no longer overflow, as at 4.5 % alone they did from 169,000 on (256 x 200,000, k = 2,000: 124 us, was 379; 3,060 kept by
// top-p: 270, was 302).  `fill` is half a deviation below the mean: at 0.6 the last k that gains was lost (1,024 x 151,936,
// k = 3,570: 672 us guessed, 806 not), at 2 batches of one wave won what those of several lost (k = 3,500: 256 rows 278 -> 258,
// 1,024 rows 565 -> 805).
void guess_for(uint32_t n, uint32_t* most, uint32_t* fill) {
    const uint32_t all = n / kChunk;
    *most = *fill = 0;
    if (n <= kList) return;  // (the whole row is listed)
    auto mean = [&](uint32_t j) { return all * std::log((all + 0.5f) / (j + 0.5f)); };
    auto deviation = [&](uint32_t j) { return all / std::sqrt(j + 0.6f); };
    uint32_t j = std::max((uint32_t)std::ceil(all * 0.045f), all > kChunks - 64 ? all - (kChunks - 64) : 0), end = all - 1;
    while (j < end) {
        const uint32_t mid = (j + end) / 2;
        if (mean(mid) + 2.5f * deviation(mid) <= (float)kList)
            end = mid;
        else
            j = mid + 1;
    }
    *most = all - j;
    *fill = (uint32_t)std::fmax(0.0f, mean(j) - 0.5f * deviation(j));
}

template <typename T>
int launch(const Args& g, uint32_t rows, cudaStream_t s) {
    int dev = 0;
    static std::atomic<int> sms[kMaxDevices];  // (every thread that fills an entry writes the same value)
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices)
        return lrs_call_error(LRS_E_CUDA, "lrs_draw_device: no current device");
    auto* kernel = draw_kernel<T>;
    if (sms[dev] == 0) {
        int count = 0;
        cudaError_t e = cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, dev);
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     (int)shared_bytes<T>(LRS_DRAW_MAX_VOCAB));
        if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return lrs_call_error(LRS_E_CUDA, "lrs_draw_device: %s", cudaGetErrorString(e));
        sms[dev] = count;
    }
    // CTAs a row: as many as give two an SM (three fit; with four the clusters' packing cost more than it gave:
    // 64 x 151,936 in 41 us and not 25), no more than give each warp a tile.  So rows above 148 have one each: with
    // two, 256 x 151,936 under the default filters took 81 us and not 52, unfiltered 89 and not 80.
    const uint32_t tiles = (g.n + 15 + kTile - 1) / kTile;
    uint32_t ctas = 1;
    while (ctas < kMaxCluster && (uint64_t)rows * ctas * 2 <= 2 * (uint64_t)sms[dev].load() && ctas * kWarps < tiles) ctas *= 2;
    // Batches of several waves go over the rows twice, the heavy rows first, so that no such row is among the last
    // to start: 1,024 x 151,936 with mixed filters in 162 us and not 193 (graph replays on one input).  The CTAs that find
    // their row in the other half leave at once.  (With one wave all start together: the second half would only cost.  Three
    // CTAs an SM hold up to n = 640,000; of longer rows, whose maxima and sums take more shared memory, a wave is smaller, and
    // batches of 149 or 297 rows up to three an SM keep the order of their rows.)
    const bool waves = ctas == 1 && rows > 3 * (uint32_t)sms[dev].load();
    Args args = g;
    args.twice = waves ? rows : 0;
    static thread_local uint32_t known[3];  // n, most, fill of the thread's last call (0.4 us)
    if (known[0] != g.n) guess_for(g.n, &known[1], &known[2]), known[0] = g.n;
    args.most = known[1], args.fill = known[2];
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(waves ? 2 * rows : rows * ctas);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = shared_bytes<T>(g.n);
    cfg.stream = s;
    cudaLaunchAttribute at[2] = {};
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = ctas, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeClusterSchedulingPolicyPreference;
    at[1].val.clusterSchedulingPolicyPreference = cudaClusterSchedulingPolicySpread;
    cfg.attrs = at;
    cfg.numAttrs = ctas > 1 ? 2 : 0;
    return launched("lrs_draw_device", cudaLaunchKernelEx(&cfg, kernel, args));
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
    const Args g{d_logits, ld, d_params, d_uniform, d_tokens, d_probs, d_kept, d_status, n, 0, 0, 0};
    const cudaStream_t s = (cudaStream_t)stream;
    return dtype == LRS_F32 ? launch<float>(g, rows, s) : dtype == LRS_BF16 ? launch<__nv_bfloat16>(g, rows, s) : launch<__half>(g, rows, s);
}
