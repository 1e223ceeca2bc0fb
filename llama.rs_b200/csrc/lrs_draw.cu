// lrs_draw.cu — draws from given uniforms with temperature, top-k, top-p and min-p (sm_100a).
//
// The definition (include/llamars_sampler.h) is over the real numbers.  Every weight that decides
// w = 2^((x - M) c), c = log2(e) / T, and every sum of them is held in 64 bits, so that a token
// differs from the real-number one only where u falls within about 1e-13 of a step of the
// distribution function.
//
// A row is one cluster of CTAs (one CTA for batches, up to 16 for a few rows), each with a slice of
// its tiles of 1024 elements; nothing is kept outside shared memory.
//   1. One pass over the logits: the maximum of every 16-byte-by-32-lane chunk and, where the whole
//      row's mass Z is asked for, the tile's sum of weights, all written to the first CTA (over
//      distributed shared memory).  With filters the sums are 32-bit ones, good to kApprox = 2^-20.
//   2. Few survivors (the first CTA): the k-th largest chunk maximum is a lower bound of the k-th
//      largest logit; maxima whose mass reaches top_p Z bound the nucleus; min-p bounds directly.
//      The chunks that reach the bound are read again, what reaches it goes to a list, the list is
//      sorted and cut; top-p's cut is taken at both ends of Z's error, and Z is summed again in 64
//      bits in the rare case that they differ.  The token comes from the kept list in index order.
//   3. Many survivors (no bound, or a list that overflows; all CTAs): histograms of count and mass
//      over the integer order of the logits narrow the cut to a bracket that fits the list, a last
//      pass sums what lies above it by tile and lists the bracket, and the token is found by tile,
//      then inside one tile.  Without any filter step 1 sums in 64 bits and goes there directly.
#include <cooperative_groups.h>

#include <cmath>

#include "lrs_ops.cuh"

namespace {

using namespace lrs;
namespace cg = cooperative_groups;

constexpr uint32_t kThreads = 512;
constexpr uint32_t kWarps = kThreads / 32;
constexpr uint32_t kTile = 1024;       // elements of a tile, 32 a lane
constexpr uint32_t kList = 4096;       // candidates that are sorted
constexpr uint32_t kChunks = 2048;     // chunks that are read again for them
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
// Chebyshev nodes on [-1/2, 1/2], 3.7e-14 off at most and exact at 0; 0 below 2^-1000.
__device__ __forceinline__ double power2(double y) {
    const double magic = 0x1.8p52;
    const double t = y + magic, f = y - (t - magic);
    double p = 0x1.b63880a30e9ffp-24;
    p = fma(p, f, 0x1.63d136366db24p-20);
    p = fma(p, f, 0x1.ffcb9515a8016p-17);
    p = fma(p, f, 0x1.4308ac85aa947p-13);
    p = fma(p, f, 0x1.5d87fe86fe88ep-10);
    p = fma(p, f, 0x1.3b2ab7181b755p-7);
    p = fma(p, f, 0x1.c6b08d7047e52p-5);
    p = fma(p, f, 0x1.ebfbdff823cedp-3);
    p = fma(p, f, 0x1.62e42fefa39efp-1);
    p = fma(p, f, 1.0);
    const uint32_t top = (uint32_t)__double2hiint(y);
    const bool gone = top > 0xC08F4000u;  // y < -1000, -inf included
    const double r = __hiloint2double(__double2hiint(p) + (__double2loint(t) << 20), __double2loint(p));
    return gone ? 0.0 : r;
}

struct Sum {
    uint32_t n;
    double lo, hi;
};

// Units of a weight of 1 in a bin's mass: the sum of n of them stays below 2^31.
__device__ __forceinline__ uint32_t mass_unit(uint32_t n) { return 1u << (__clz((n - 1) | 1) - 2); }

struct Shared {
    Sum part[kWarps];
    Sum from[kMaxCluster];       // (first CTA: the others' sums)
    float top[kWarps], tops[kMaxCluster];
    uint32_t word[kWarps];
    uint32_t order[4];           // what the first CTA has all do next: operation, upper and lower key, shift
    uint32_t count, chunks;      // entries of the lists
    uint64_t cut;
};

enum { kDone, kHistogram, kSumAbove, kGather, kGatherTies };

__device__ __forceinline__ Sum add(const Sum& a, const Sum& b) { return Sum{a.n + b.n, a.lo + b.lo, a.hi + b.hi}; }

// Sums over the CTA in one order; every thread gets the total, and the sum of the threads before it.
__device__ __noinline__ Sum block_scan(Sum v, Sum* before, Shared& sh) {
    const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    Sum inc = v;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        Sum p{__shfl_up_sync(kAll, inc.n, o), __shfl_up_sync(kAll, inc.lo, o), __shfl_up_sync(kAll, inc.hi, o)};
        if (lane >= o) inc = add(p, inc);
    }
    __syncthreads();
    if (lane == 31) sh.part[warp] = inc;
    __syncthreads();
    Sum t{0, 0.0, 0.0}, w{0, 0.0, 0.0};
    for (uint32_t i = 0; i < kWarps; ++i) {
        if (i == warp) w = t;
        t = add(t, sh.part[i]);
    }
    if (before) {
        Sum p{__shfl_up_sync(kAll, inc.n, 1), __shfl_up_sync(kAll, inc.lo, 1), __shfl_up_sync(kAll, inc.hi, 1)};
        *before = lane ? add(w, p) : w;
    }
    return t;
}

__device__ __noinline__ uint32_t block_min(uint32_t v, Shared& sh) {
    v = __reduce_min_sync(kAll, v);
    __syncthreads();
    if (threadIdx.x % 32 == 0) sh.word[threadIdx.x / 32] = v;
    __syncthreads();
    for (uint32_t i = 0; i < kWarps; ++i) v = min(v, sh.word[i]);
    return v;
}

// Bitonic sort of list[0 .. 2^m) (2^m >= count, entries from count on given `pad` here), ascending or
// descending.  Steps whose pairs stay within a warp's 64 entries need no barrier of the CTA.
template <bool DESC>
__device__ __noinline__ void sort(uint64_t* list, uint32_t count) {
    uint32_t size = 2;
    while (size < count) size *= 2;
    for (uint32_t i = count + threadIdx.x; i < size; i += kThreads) list[i] = DESC ? 0ull : ~0ull;
    __syncthreads();
    for (uint32_t m = 2; m <= size; m *= 2)
        for (uint32_t j = m / 2; j > 0; j /= 2) {
            for (uint32_t t = threadIdx.x; t < size / 2; t += kThreads) {
                const uint32_t i = 2 * t - (t & (j - 1));
                const uint64_t a = list[i], b = list[i + j];
                if ((a > b) != (((i & m) != 0) ^ DESC)) list[i] = b, list[i + j] = a;
            }
            if (j > 32 || (j == 1 && m >= 64) || size / 2 > kThreads)
                __syncthreads();
            else
                __syncwarp();
        }
    __syncthreads();
}

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
};

// The row as this call sees it: element i at base[i + skew], base on a 16-byte boundary.
template <typename T>
struct RowView {
    static constexpr uint32_t kVec = 16 / sizeof(T), kChunk = 32 * kVec, kPer = kTile / kChunk;
    const T* base;
    uint32_t skew, end;  // elements are base[skew .. end)

    // V consecutive elements from position j (a multiple of V); -inf outside the row
    __device__ __forceinline__ void vec(uint32_t j, float* v) const {
        if (j >= skew && j + kVec <= end) {
            float x[kVec];
            unpack(__ldg(reinterpret_cast<const uint4*>(base + j)), x, base);
#pragma unroll
            for (uint32_t i = 0; i < kVec; ++i) v[i] = x[i];
        } else {
#pragma unroll
            for (uint32_t i = 0; i < kVec; ++i) v[i] = j + i >= skew && j + i < end ? to_float<T>(base[j + i]) : -INFINITY;
        }
    }
    __device__ __forceinline__ void tile(uint32_t t, float (&v)[32]) const {
        const uint32_t j = t * kTile + threadIdx.x % 32 * kVec;
        if (t * kTile >= skew && t * kTile + kTile <= end) {
            uint4 r[kPer];
#pragma unroll
            for (uint32_t c = 0; c < kPer; ++c) r[c] = __ldg(reinterpret_cast<const uint4*>(base + j + c * kChunk));
#pragma unroll
            for (uint32_t c = 0; c < kPer; ++c) {
                float x[kVec];
                unpack(r[c], x, base);
#pragma unroll
                for (uint32_t i = 0; i < kVec; ++i) v[c * kVec + i] = x[i];
            }
        } else {
#pragma unroll
            for (uint32_t c = 0; c < kPer; ++c) vec(j + c * kChunk, v + c * kVec);
        }
    }
};

// Weights relative to a maximum.
struct Weigh {
    double max, c;
    __device__ __forceinline__ double operator()(float x) const { return power2(((double)x - max) * c); }
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

// One operation of the first CTA's over this CTA's slice of the row: keys from `hi` up are summed, those
// of [lo, hi) counted by bin, listed, or counted by tile.
template <typename T>
struct Slice {
    RowView<T> row;
    uint32_t t0, t1, n;  // tiles of the slice, elements of the row
    double c;
    uint8_t* dynamic;    // (as the kernel lays it out)
    double* first_sum;
    float* first_max;
};

template <typename T>
__device__ __noinline__ void perform(const Slice<T>& z, float max, Shared& sh) {
    using View = RowView<T>;
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const uint32_t op = sh.order[0], hi = sh.order[1], lo = sh.order[2], shift = sh.order[3];
    uint32_t* bin_n = reinterpret_cast<uint32_t*>(z.dynamic);
    uint32_t* bin_w = bin_n + kBins;
    uint64_t* first_list = cluster.map_shared_rank(reinterpret_cast<uint64_t*>(z.dynamic), 0);
    uint32_t* first_count = cluster.map_shared_rank(&sh.count, 0);
    const Weigh weigh{(double)max, z.c};
    const float cf = (float)z.c, scale = (float)mass_unit(z.n);
    Sum s{0, 0.0, 0.0};  // elements from hi up: count and mass; mass of all (histograms)
    if (op == kHistogram) {
        for (uint32_t i = threadIdx.x; i < 2 * kBins; i += kThreads) bin_n[i] = 0;
        __syncthreads();
    }
    for (uint32_t t = z.t0 + warp; t < z.t1; t += kWarps) {
        float v[32];
        z.row.tile(t, v);
        double above = 0.0;
        if (op == kHistogram) {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const uint32_t key = key_of(v[i]);
                const double w = weigh(v[i]);
                s.hi += w;
                if (key >= hi) {
                    s.lo += w, ++s.n;
                } else if (key >= lo) {
                    const uint32_t b = (hi - 1 - key) >> shift;
                    const float edge = ceilf((value_of(hi - 1 - (b << shift)) - max) * cf);
                    float e;
                    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"((v[i] - max) * cf - edge));
                    atomicAdd(&bin_n[b], 1u);
                    atomicAdd(&bin_w[b], __float2uint_rn(fminf(e, 2.0f) * scale));
                }
            }
            continue;
        }
        uint32_t ties = 0;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const uint32_t key = key_of(v[i]);
            if (key >= hi) above += weigh(v[i]), ++s.n;
            ties += key >= lo && key < hi;
        }
        s.lo += above;
        if (op == kSumAbove) continue;
        above = warp_sum(above);
        if (lane == 0) z.first_sum[t] = above;
        if (op == kGatherTies) {
            ties = __reduce_add_sync(kAll, ties);
            if (lane == 0) reinterpret_cast<uint32_t*>(z.first_max)[t] = ties;
        } else {
            // the lane's place in the list, then its elements in turn
            uint32_t inc = ties;
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const uint32_t q = __shfl_up_sync(kAll, inc, o);
                if (lane >= o) inc += q;
            }
            const uint32_t all = __shfl_sync(kAll, inc, 31);
            if (all == 0) continue;
            uint32_t at = 0;
            if (lane == 0) at = atomicAdd(first_count, all);
            at = __shfl_sync(kAll, at, 0) + inc - ties;
            if (ties == 0) continue;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const uint32_t key = key_of(v[i]);
                if (key < lo || key >= hi) continue;
                const uint32_t index = t * kTile + i / View::kVec * View::kChunk + lane * View::kVec + i % View::kVec - z.row.skew;
                if (at < kList) first_list[at] = (uint64_t)key << 32 | ~index;
                ++at;
            }
        }
    }
    s = block_scan(s, nullptr, sh);
    if (threadIdx.x == 0) *cluster.map_shared_rank(&sh.from[cluster.block_rank()], 0) = s;
    if (cluster.num_blocks() > 1)
        cluster.sync();
    else
        __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) draw_kernel(const Args g) {
    extern __shared__ __align__(16) uint8_t dynamic[];
    __shared__ Shared sh;
    using View = RowView<T>;
    constexpr uint32_t kPer = View::kPer, kVec = View::kVec, kChunk = View::kChunk;
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t ctas = cluster.num_blocks(), rank = cluster.block_rank();
    const uint32_t r = blockIdx.x / ctas, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    auto all_sync = [&] {
        if (ctas > 1)
            cluster.sync();
        else
            __syncthreads();
    };

    const lrs_draw_params p = g.params[r];
    const bool greedy = p.temperature <= 0.0f;
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
    View row;
    {
        const T* x = reinterpret_cast<const T*>(g.logits) + r * g.ld;
        row.skew = (uint32_t)((uintptr_t)x % 16 / sizeof(T));
        row.base = x - row.skew;
        row.end = n + row.skew;
    }
    const uint32_t tiles = (row.end + kTile - 1) / kTile, chunks = tiles * kPer;
    const uint32_t each = (tiles + ctas - 1) / ctas, t0 = min(tiles, rank * each), t1 = min(tiles, t0 + each);

    uint64_t* list = reinterpret_cast<uint64_t*>(dynamic);                 // kList entries, or
    uint32_t* bin_n = reinterpret_cast<uint32_t*>(dynamic);                // kBins counts and
    uint32_t* bin_w = bin_n + kBins;                                       // kBins masses
    uint32_t* again = reinterpret_cast<uint32_t*>(list + kList);           // kChunks chunk numbers
    double* tile_sum = reinterpret_cast<double*>(again + kChunks);         // a tile's
    float* chunk_max = reinterpret_cast<float*>(tile_sum + (tiles + 1) / 2 * 2);
    double* first_sum = cluster.map_shared_rank(tile_sum, 0);
    float* first_max = cluster.map_shared_rank(chunk_max, 0);

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
        float tile_top = -INFINITY, mine = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < kPer; ++i) {
            float m = v[i * kVec];
#pragma unroll
            for (uint32_t e = 1; e < kVec; ++e) m = max_nan(m, v[i * kVec + e]);
            m = warp_max_nan(m);
            if (lane == i) mine = m;
            tile_top = max_nan(tile_top, m);
        }
        if (lane < kPer) first_max[t * kPer + lane] = mine;
        top = max_nan(top, tile_top);
        if (!(by_mass || whole) || greedy) continue;
        double s = 0.0;
        if (isfinite(tile_top)) {
            if (!whole && rough.fits(tile_top)) {
                s = warp_sum((double)rough.sum(v, tile_top));
            } else {
                const Weigh w{(double)tile_top, c};
#pragma unroll
                for (int i = 0; i < 32; ++i) s += w(v[i]);
                s = warp_sum(s);
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
            float v[kVec];
            const uint32_t j = at * kChunk + lane * kVec;
            row.vec(j, v);
            uint32_t index = kAll;
#pragma unroll
            for (int e = (int)kVec - 1; e >= 0; --e)
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

    // Sorted candidates (below `base` kept elements): how many of them are kept.
    auto cut_list = [&](uint32_t count, const Sum& base, double reach_a, double reach_b, uint32_t* at_b) {
        const uint32_t per = (count + kThreads - 1) / kThreads;
        const uint32_t i0 = min(count, threadIdx.x * per), i1 = min(count, i0 + per);
        Sum s{0, 0.0, 0.0}, before;
        for (uint32_t i = i0; i < i1; ++i) s.lo += weigh(value_of((uint32_t)(list[i] >> 32)));
        block_scan(s, &before, sh);
        double run = base.lo + before.lo;
        uint32_t a = 0, b = 0;
        for (uint32_t i = i0; i < i1; ++i) {
            const double w = weigh(value_of((uint32_t)(list[i] >> 32)));
            const bool in = base.n + i < k && w >= (double)p.min_p;
            a += in && run < reach_a;
            b += in && run < reach_b;
            run += w;
        }
        const Sum both = block_scan(Sum{a | b << 16, 0.0, 0.0}, nullptr, sh);  // (at most 4096 each)
        *at_b = both.n >> 16;
        return both.n & 0xFFFFu;
    };
    // The kept elements of the list, re-keyed and sorted by index.
    auto by_index = [&](uint32_t count) {
        for (uint32_t i = threadIdx.x; i < count; i += kThreads) {
            const uint64_t e = list[i];
            list[i] = (uint64_t)~(uint32_t)e << 32 | e >> 32;
        }
        __syncthreads();
        sort<false>(list, count);
    };

    if (!whole) {
        // ---- 2. few survivors ----
        uint32_t bound = kLowest;
        if (p.min_p > 0.0f) {
            const double below = log2((double)p.min_p) / c;
            const double x = (double)top + below - (fabs((double)top) - below) * 1e-12;
            bound = max(bound, key_of(__double2float_rd(x)));
        }
        // the largest key at which the chunk maxima alone fill top_k or top_p (no need to find it to the
        // last bit: a few chunks more cost less than the steps)
        auto filled = [&](uint32_t key, uint32_t* count) {
            Sum s{0, 0.0, 0.0};
            for (uint32_t i = threadIdx.x; i < chunks; i += kThreads) {
                const float m = chunk_max[i];
                if (key_of(m) >= key) {
                    ++s.n;
                    if (by_mass) s.lo += weigh(m);
                }
            }
            s = block_scan(s, nullptr, sh);
            *count = s.n;
            return s.n >= k || s.lo >= reach_hi;
        };
        uint32_t reaching;
        if (filled(bound, &reaching)) {
            uint32_t lo = bound, hi = key_of(top) + 1;
            while (hi - lo > 1 && reaching > (k < chunks ? k + 32 : 64)) {
                const uint32_t mid = lo + (hi - lo) / 2;
                uint32_t count;
                if (filled(mid, &count))
                    lo = mid, reaching = count;
                else
                    hi = mid;
            }
            bound = lo;
        }
        __syncthreads();
        if (threadIdx.x == 0) sh.count = 0, sh.chunks = 0;
        __syncthreads();
        if (reaching <= kChunks) {
            for (uint32_t i = threadIdx.x; i < chunks; i += kThreads)
                if (key_of(chunk_max[i]) >= bound) again[atomicAdd(&sh.chunks, 1u)] = i;
            __syncthreads();
            constexpr uint32_t kAtOnce = 16 / kVec;
            for (uint32_t i = warp * kAtOnce; i < reaching; i += kWarps * kAtOnce) {
                float v[kAtOnce][kVec];
#pragma unroll
                for (uint32_t q = 0; q < kAtOnce; ++q)
                    if (i + q < reaching) row.vec(again[i + q] * kChunk + lane * kVec, v[q]);
#pragma unroll
                for (uint32_t q = 0; q < kAtOnce; ++q) {
                    if (i + q >= reaching) break;
                    const uint32_t j = again[i + q] * kChunk + lane * kVec - row.skew;
#pragma unroll
                    for (uint32_t e = 0; e < kVec; ++e) {
                        const uint32_t key = key_of(v[q][e]);
                        const uint32_t vote = __ballot_sync(kAll, key >= bound);
                        if (vote == 0) continue;
                        uint32_t at = 0;
                        if (lane == 0) at = atomicAdd(&sh.count, __popc(vote));
                        at = __shfl_sync(kAll, at, 0) + __popc(vote & ((1u << lane) - 1));
                        if (key >= bound && at < kList) list[at] = (uint64_t)key << 32 | ~(j + e);
                    }
                }
            }
            __syncthreads();
            const uint32_t count = sh.count;
            if (count <= kList) {
                sort<true>(list, count);
                uint32_t other;
                uint32_t keep = cut_list(count, Sum{0, 0.0, 0.0}, reach_lo, reach_hi, &other);
                if (keep != other) {  // Z's error decides: the row's mass again, in 64 bits
                    Sum s{0, 0.0, 0.0};
                    for (uint32_t t = warp; t < tiles; t += kWarps) {
                        float v[32];
                        row.tile(t, v);
#pragma unroll
                        for (int i = 0; i < 32; ++i) s.lo += weigh(v[i]);
                    }
                    z = block_scan(s, nullptr, sh).lo;
                    keep = cut_list(count, Sum{0, 0.0, 0.0}, top_p * z, top_p * z, &other);
                }
                by_index(keep);
                const uint32_t per = (keep + kThreads - 1) / kThreads;
                const uint32_t i0 = min(keep, threadIdx.x * per), i1 = min(keep, i0 + per);
                Sum s{0, 0.0, 0.0}, before;
                for (uint32_t i = i0; i < i1; ++i) s.lo += weigh(value_of((uint32_t)list[i]));
                const double mass = block_scan(s, &before, sh).lo, target = (double)u * mass;
                uint32_t found = kAll;
                double run = before.lo;
                for (uint32_t i = i0; i < i1; ++i) {
                    run += weigh(value_of((uint32_t)list[i]));
                    if (run > target) {
                        found = i;
                        break;
                    }
                }
                found = block_min(found, sh);
                if (threadIdx.x == 0) {
                    if (found == kAll)  // (two orders of a sum: the last weight, when none passes the target)
                        for (found = keep - 1; found > 0 && weigh(value_of((uint32_t)list[found])) == 0.0;) --found;
                    const uint64_t e = list[found];
                    finish(LRS_OK, (uint32_t)(e >> 32), weigh(value_of((uint32_t)e)) / mass, keep);
                }
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
        if (by_mass) {  // what is lighter than (1 - top_p) Z / n is left out even if every element is
            const double below = log2((1.0 - top_p) * z * (1.0 - 2.0 * kApprox) / n) / c;
            lo = max(lo, key_of(__double2float_rd((double)top + below - (fabs((double)top) + fabs(below)) * 1e-12)));
        }
        if (hi <= lo) lo = hi - 1;
        uint32_t inside = kAll;  // elements of [lo, hi)
        Sum base{0, 0.0, 0.0};
        double reach = INFINITY;
        for (int round = 0; round < 3 && inside > kList && (hi - lo > 1 || round == 0); ++round) {
            const uint32_t range = hi - lo;
            const uint32_t bits = 32 - __clz(range - 1 | 1);
            const uint32_t shift = bits > 12 ? bits - 12 : 0;
            command(kHistogram, hi, lo, shift);
            perform(slice, top, sh);
            base = total();
            if (by_mass) reach = top_p * base.hi;
            for (uint32_t q = 1; q < ctas; ++q) {
                const uint32_t* other = cluster.map_shared_rank(bin_n, q);
                for (uint32_t i = threadIdx.x; i < 2 * kBins; i += kThreads) bin_n[i] += other[i];
            }
            __syncthreads();
            // where the cut may lie: counts are exact, masses within their rounding (half a unit an
            // element, and the 32-bit power)
            constexpr uint32_t kEach = kBins / kThreads;
            const float cf = (float)c;
            const double unit = 1.0 / (double)mass_unit(n);
            auto mass = [&](uint32_t b, bool upper) {
                const uint32_t w = bin_w[b], m = bin_n[b];
                if (m == 0 || !by_mass) return 0.0;
                const float y = (value_of(hi - 1 - (b << shift)) - top) * cf;
                const double err = 0x1p-20 * (2.0 + fabs((double)y));
                const double s = unit * power2(fmax((double)ceilf(y), -2000.0));
                return upper ? ((double)w + m) * s * (1.0 + err) : fmax(0.0, ((double)w - m) * s * (1.0 - err));
            };
            Sum s{0, 0.0, 0.0}, before;
            for (uint32_t i = 0; i < kEach; ++i) {
                const uint32_t b = threadIdx.x * kEach + i;
                s.n += bin_n[b], s.lo += mass(b, false), s.hi += mass(b, true);
            }
            block_scan(s, &before, sh);
            Sum run{base.n + before.n, base.lo + before.lo, base.lo + before.hi};
            uint32_t a = kBins - 1, z1 = kBins - 1;
            for (uint32_t i = 0; i < kEach; ++i) {
                const uint32_t b = threadIdx.x * kEach + i;
                run.n += bin_n[b], run.lo += mass(b, false), run.hi += mass(b, true);
                if ((run.n >= k || run.hi >= reach) && b < a) a = b;
                if ((run.n >= k || run.lo >= reach) && b < z1) z1 = b;
            }
            a = block_min(a, sh), z1 = block_min(z1, sh);
            const uint32_t last = (range - 1) >> shift;
            a = min(a, last), z1 = min(z1, last);
            Sum in{0, 0.0, 0.0};
            for (uint32_t b = a + threadIdx.x; b <= z1; b += kThreads) in.n += bin_n[b];
            inside = block_scan(in, nullptr, sh).n;
            const uint32_t from = hi;
            hi = from - (a << shift);
            lo = max(lo, from - min(from, (z1 + 1) << shift));
        }
        // (histograms that do not settle, as with a mass far below their unit: halves, summed exactly)
        while (inside > kList && hi - lo > 1) {
            const uint32_t mid = lo + (hi - lo) / 2;
            command(kSumAbove, mid, mid, 0);
            perform(slice, top, sh);
            const Sum s = total();
            if (s.n >= k || s.lo >= reach) {
                lo = mid;
            } else {
                hi = mid;
            }
            command(kSumAbove, hi, hi, 0);
            perform(slice, top, sh);
            const uint32_t above = total().n;
            command(kSumAbove, lo, lo, 0);
            perform(slice, top, sh);
            inside = total().n - above;
        }
        const bool ties = inside > kList;  // (of one key)
        __syncthreads();
        if (threadIdx.x == 0) sh.count = 0;
        command(ties ? kGatherTies : kGather, hi, lo, 0);
        perform(slice, top, sh);
        const Sum above = total();
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
            sort<true>(list, count);
            uint32_t other;
            const uint32_t keep = cut_list(count, above, reach, reach, &other);
            cut = keep ? list[keep - 1] : (uint64_t)hi << 32;
            kept = above.n + keep;
            __syncthreads();
            by_index(keep);
            for (uint32_t t = threadIdx.x; t < tiles; t += kThreads) {
                const uint32_t from = t * kTile < row.skew ? 0 : t * kTile - row.skew;  // the tile's first index
                uint32_t a = 0, b = keep;
                while (a < b) {
                    const uint32_t mid = (a + b) / 2;
                    if ((uint32_t)(list[mid] >> 32) < from)
                        a = mid + 1;
                    else
                        b = mid;
                }
                double w = tile_sum[t];
                for (; a < keep && (uint32_t)(list[a] >> 32) < (t + 1) * kTile - row.skew; ++a)
                    w += weigh(value_of((uint32_t)list[a]));
                tile_sum[t] = w;
            }
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
    for (uint32_t t = i0; t < i1; ++t) {
        if (tile_sum[t] > 0.0) heavy = t + 1;
        if (at == kAll && run + tile_sum[t] > target) at = t, base = run;
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
    if (warp == 0) {
        double before_v = sh.part[0].lo;
        const uint32_t quota = tie_keep ? reinterpret_cast<uint32_t*>(chunk_max)[tile] : 0;
        uint32_t seen = 0, token = kAll, final = kAll;
        double w_token = 0.0, w_final = 0.0;
        for (uint32_t i = 0; i < kPer && token == kAll; ++i) {
            float v[kVec];
            double w[kVec], sum = 0.0;
            const uint32_t j = tile * kTile + i * kChunk + lane * kVec;
            row.vec(j, v);
            uint32_t tied = 0;
#pragma unroll
            for (uint32_t e = 0; e < kVec; ++e) tied += tie_keep && key_of(v[e]) == tie_key;
            uint32_t rank_before = tied;
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const uint32_t q = __shfl_up_sync(kAll, rank_before, o);
                if (lane >= o) rank_before += q;
            }
            const uint32_t chunk_ties = __shfl_sync(kAll, rank_before, 31);
            uint32_t q = seen + rank_before - tied;
            seen += chunk_ties;
#pragma unroll
            for (uint32_t e = 0; e < kVec; ++e) {
                const uint32_t key = key_of(v[e]);
                const uint64_t entry = (uint64_t)key << 32 | ~(j + e - row.skew);
                bool in = key >= kLowest && entry >= cut;
                if (tie_keep && key == tie_key) in = q++ < quota;
                w[e] = in ? weigh(v[e]) : 0.0;
                sum += w[e];
            }
            double inc = sum;
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const double d = __shfl_up_sync(kAll, inc, o);
                if (lane >= o) inc += d;
            }
            double here = before_v + (inc - sum);
            uint32_t mine = kAll, mine_last = 0;
            double w_mine = 0.0, w_last = 0.0;
#pragma unroll
            for (uint32_t e = 0; e < kVec; ++e) {
                here += w[e];
                if (w[e] > 0.0) {
                    mine_last = j + e - row.skew + 1, w_last = w[e];
                    if (mine == kAll && here > target && before_v < INFINITY) mine = j + e - row.skew, w_mine = w[e];
                }
            }
            const uint32_t first = __reduce_min_sync(kAll, mine);
            if (first != kAll) {
                const uint32_t who = __ffs(__ballot_sync(kAll, mine == first)) - 1;
                token = first, w_token = __shfl_sync(kAll, w_mine, who);
            }
            const uint32_t end = __reduce_max_sync(kAll, mine_last);
            if (end) {
                const uint32_t who = __ffs(__ballot_sync(kAll, mine_last == end)) - 1;
                final = end - 1, w_final = __shfl_sync(kAll, w_last, who);
            }
            before_v += __shfl_sync(kAll, inc, 31);
        }
        if (token == kAll) token = final, w_token = w_final;
        if (lane == 0) finish(LRS_OK, token, w_token / mass, kept);
    }
}

constexpr int kMaxDevices = 64;

template <typename T>
size_t shared_bytes(uint32_t n) {
    const uint32_t tiles = (n + 15 + kTile - 1) / kTile;
    return kList * 8 + kChunks * 4 + (tiles + 1) / 2 * 2 * 8 + (size_t)tiles * RowView<T>::kPer * 4;
}

template <typename T>
int launch(const Args& g, uint32_t rows, cudaStream_t s) {
    int dev = 0;
    static int sms[kMaxDevices];  // (every thread that fills an entry writes the same value)
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
    // CTAs a row: as many as fill two an SM, no more than give each warp a tile
    const uint32_t tiles = (g.n + 15 + kTile - 1) / kTile;
    uint32_t ctas = 1;
    while (ctas < kMaxCluster && (uint64_t)rows * ctas * 2 <= 2 * (uint64_t)sms[dev] && ctas * kWarps < tiles) ctas *= 2;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(rows * ctas);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = shared_bytes<T>(g.n);
    cfg.stream = s;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = ctas, at.val.clusterDim.y = 1, at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, g);
    return e == cudaSuccess ? LRS_OK : lrs_call_error(LRS_E_CUDA, "lrs_draw_device: launch failed: %s", cudaGetErrorString(e));
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
    const Args g{d_logits, ld, d_params, d_uniform, d_tokens, d_probs, d_kept, d_status, n};
    const cudaStream_t s = (cudaStream_t)stream;
    return dtype == LRS_F32 ? launch<float>(g, rows, s) : dtype == LRS_BF16 ? launch<__nv_bfloat16>(g, rows, s) : launch<__half>(g, rows, s);
}
