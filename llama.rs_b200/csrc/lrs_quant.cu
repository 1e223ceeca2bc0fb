// lrs_quant.cu — e4m3 codes with one f32 scale per block (sm_100a): lrs_quantize_rows (1 x 128,
// activations) and lrs_quantize_blocks (128 x 128, weights).
//
//   m = max |x| over the block,  s = max(m / 448, 2^-126),  code = e4m3(x * (1 / s))
//
// 448 is e4m3's largest value, so no code saturates; 2^-126 keeps 1 / s finite (an all-zero block
// gets codes 0).  Each step is one f32 operation, so a program that follows the three lines gets
// the same bits.  A NaN travels through the max into the scale; an infinity makes s infinite.
//
// Bound: HBM (one read of x, one write of a byte an element).  A block's elements stay in
// registers between the max and the codes, so x is read once.
#include "lrs_ops.cuh"

namespace {

using namespace lrs;

constexpr uint32_t kBlock = 128;
constexpr uint32_t kThreads = 256;

__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

__device__ __forceinline__ float scale_of(float m) { return max_nan(__fdiv_rn(m, 448.0f), 1.17549435e-38f); }

__device__ __forceinline__ uint32_t bits_of(float v) { return __float_as_uint(v); }
__device__ __forceinline__ uint32_t bits_of(__nv_bfloat16 v) { return __bfloat16_as_ushort(v); }
__device__ __forceinline__ uint32_t bits_of(__half v) { return __half_as_ushort(v); }

// The 16 bytes of a row that start at column c (on a 16-byte boundary), zeros outside the row: one
// load where they are all inside.
template <typename T>
__device__ __forceinline__ uint4 load_aligned(const T* row, int32_t c, uint32_t k) {
    constexpr int32_t kVec = 16 / sizeof(T), kEach = kVec / 4;
    if (c >= 0 && c + kVec <= (int32_t)k) return __ldg(reinterpret_cast<const uint4*>(row + c));
    uint32_t w[4];
#pragma unroll
    for (int32_t i = 0; i < 4; ++i) {
        w[i] = 0;
#pragma unroll
        for (int32_t j = 0; j < kEach; ++j) {
            const int32_t e = c + i * kEach + j;
            if (e >= 0 && e < (int32_t)k) w[i] |= bits_of(row[e]) << (16 * j);
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// The same for any alignment of the row: the two aligned 16 bytes around it, shifted (the second load
// finds its neighbour's line in L1).  On 109,051 x 1,001 bf16 element loads reached 1,580 GB/s, this
// 2,730.
template <bool ALIGNED, typename T>
__device__ __forceinline__ uint4 load(const T* row, uint32_t c, uint32_t k) {
    if constexpr (ALIGNED) return load_aligned(row, (int32_t)c, k);
    const uint32_t skew = (uint32_t)((uintptr_t)row % 16);  // (of the whole group: c is a multiple of 16 bytes)
    const int32_t at = (int32_t)c - (int32_t)(skew / sizeof(T));
    const uint4 a = load_aligned(row, at, k);
    if (skew == 0) return a;
    const uint4 b = load_aligned(row, at + (int32_t)(16 / sizeof(T)), k);
    const bool two = skew & 8, one = skew & 4;
    uint32_t w[7] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z};
    const uint32_t last = b.w;
    if (two) w[0] = w[2], w[1] = w[3], w[2] = w[4], w[3] = w[5], w[4] = w[6], w[5] = last;
    if (one) w[0] = w[1], w[1] = w[2], w[2] = w[3], w[3] = w[4], w[4] = w[5];
    const uint32_t bits = skew % 4 * 8;
    return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits),
                      __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits));
}

template <int VEC>
__device__ __forceinline__ void store(uint8_t* row, uint32_t c, uint32_t k, bool wide, const float (&x)[VEC], float inv) {
    uint32_t w[VEC / 4];
#pragma unroll
    for (int i = 0; i < VEC; i += 4)
        w[i / 4] = e4m3x2(x[i] * inv, x[i + 1] * inv) | e4m3x2(x[i + 2] * inv, x[i + 3] * inv) << 16;
    if (wide && c + VEC <= k) {
        if constexpr (VEC == 8)
            *reinterpret_cast<uint2*>(row + c) = make_uint2(w[0], w[1]);
        else
            *reinterpret_cast<uint32_t*>(row + c) = w[0];
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (c + i < k) row[c + i] = (uint8_t)(w[i / 4] >> (8 * (i % 4)));
    }
}

// The largest magnitude of 16 bytes and m, a NaN kept.  The elements stay packed: half the registers of
// unpacked 16-bit ones, so twice the loads in flight (2,160 -> 6,110 GB/s on 151,936 x 1,024 bf16).
__device__ __forceinline__ float amax(const uint4& v, float m, const float*) {
    m = max_nan(m, fabsf(__uint_as_float(v.x)));
    m = max_nan(m, fabsf(__uint_as_float(v.y)));
    m = max_nan(m, fabsf(__uint_as_float(v.z)));
    return max_nan(m, fabsf(__uint_as_float(v.w)));
}
__device__ __forceinline__ float amax(const uint4& v, float m, const __nv_bfloat16*) {
    auto part = [](uint32_t u) {
        u &= 0x7FFF7FFFu;
        return *reinterpret_cast<__nv_bfloat162*>(&u);
    };
    const __nv_bfloat162 h = __hmax2_nan(__hmax2_nan(part(v.x), part(v.y)), __hmax2_nan(part(v.z), part(v.w)));
    return max_nan(m, max_nan(__low2float(h), __high2float(h)));
}
__device__ __forceinline__ float amax(const uint4& v, float m, const __half*) {
    auto part = [](uint32_t u) {
        u &= 0x7FFF7FFFu;
        return *reinterpret_cast<__half2*>(&u);
    };
    const __half2 h = __hmax2_nan(__hmax2_nan(part(v.x), part(v.y)), __hmax2_nan(part(v.z), part(v.w)));
    return max_nan(m, max_nan(__low2float(h), __high2float(h)));
}

// A group of 128 / VEC lanes takes one block of 128 columns of kRows consecutive rows: kRows
// loads in flight a lane, and the block's kRows scales (block-major) go out in one store each of
// consecutive lanes.
constexpr int kRows = 4;
constexpr int kRowCtas = 6;

template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(kThreads, kRowCtas) quantize_rows_kernel(const T* __restrict__ x, uint32_t rows, uint32_t k,
                                                                    uint64_t ld_x, uint8_t* __restrict__ q, uint64_t ld_q,
                                                                    float* __restrict__ scale, uint64_t ld_scale,
                                                                    uint32_t blocks, bool wide) {
    constexpr uint32_t kVec = 16 / sizeof(T), kLanes = kBlock / kVec;
    const uint64_t unit = ((uint64_t)blockIdx.x * kThreads + threadIdx.x) / kLanes;
    const uint32_t lane = threadIdx.x % kLanes;
    const uint32_t b = (uint32_t)(unit % blocks);
    const uint64_t r0 = unit / blocks * kRows;
    if (r0 >= rows) return;  // (whole groups leave: the shuffles below stay within a group)
    const uint32_t c = b * kBlock + lane * kVec;
    const uint32_t mask = kLanes == 32 ? 0xFFFFFFFFu : 0xFFFFu << (threadIdx.x & 16u);
    uint4 v[kRows];
#pragma unroll
    for (int j = 0; j < kRows; ++j)
        v[j] = r0 + j < rows ? load<ALIGNED>(x + (r0 + j) * ld_x, c, k) : make_uint4(0, 0, 0, 0);
    // the rows' maxima: each exchange halves the rows a lane answers for, so that a lane's upper two
    // bits are its row in the end (5 or 6 exchanges in place of 16 or 20) and it alone divides for it
    float m[kRows];
#pragma unroll
    for (int j = 0; j < kRows; ++j) m[j] = amax(v[j], 0.0f, x);
#pragma unroll
    for (uint32_t o = kLanes / 2, h = kRows / 2; o > 0; o /= 2, h /= 2) {
        const bool upper = lane & o;
        if (h > 0) {
#pragma unroll
            for (uint32_t i = 0; i < kRows / 2; ++i)
                if (i < h) {
                    const float other = __shfl_xor_sync(mask, upper ? m[i] : m[i + h], o);
                    m[i] = max_nan(upper ? m[i + h] : m[i], other);
                }
        } else {
            m[0] = max_nan(m[0], __shfl_xor_sync(mask, m[0], o));
        }
    }
    constexpr uint32_t kShare = kLanes / kRows;  // lanes of a row's maximum
    const float s = scale_of(m[0]), inv = __frcp_rn(s);
    if (lane % kShare == 0 && r0 + lane / kShare < rows) scale[b * ld_scale + r0 + lane / kShare] = s;
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
        const float g = __shfl_sync(mask, inv, j * kShare, kLanes);
        float f[kVec];
        unpack(v[j], f, x);
        if (r0 + j < rows) store<kVec>(q + (r0 + j) * ld_q, c, k, wide, f, g);
    }
}

// One CTA takes one 128 x 128 block, eight 16-byte loads a thread.
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(16 * sizeof(T) * 8, 1024 / (16 * sizeof(T) * 8))
    quantize_blocks_kernel(const T* __restrict__ x, uint32_t rows, uint32_t k, uint64_t ld_x, uint8_t* __restrict__ q,
                           uint64_t ld_q, float* __restrict__ scale, uint64_t ld_scale, uint32_t blocks, bool wide) {
    constexpr uint32_t kVec = 16 / sizeof(T), kLanes = kBlock / kVec, kWide = 16 * sizeof(T) * 8, kStep = kWide / kLanes;
    constexpr int kN = kBlock / kStep;
    static_assert(kN == 8, "eight loads a thread");
    __shared__ float part[kWide / 32];
    const uint32_t a = blockIdx.x / blocks, b = blockIdx.x % blocks;
    const uint32_t c = b * kBlock + threadIdx.x % kLanes * kVec;
    const uint64_t r0 = (uint64_t)a * kBlock + threadIdx.x / kLanes;
    uint4 v[kN];
#pragma unroll
    for (int j = 0; j < kN; ++j)
        v[j] = r0 + j * kStep < rows ? load<ALIGNED>(x + (r0 + j * kStep) * ld_x, c, k) : make_uint4(0, 0, 0, 0);
    float m = 0.0f;
#pragma unroll
    for (int j = 0; j < kN; ++j) m = amax(v[j], m, x);
#pragma unroll
    for (uint32_t o = 16; o > 0; o /= 2) m = max_nan(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = m;
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < kWide / 32; ++w) m = max_nan(m, part[w]);
    const float s = scale_of(m), inv = __frcp_rn(s);
    if (threadIdx.x == 0) scale[a * ld_scale + b] = s;
#pragma unroll
    for (int j = 0; j < kN; ++j) {
        float f[kVec];
        unpack(v[j], f, x);
        if (r0 + j * kStep < rows) store<kVec>(q + (r0 + j * kStep) * ld_q, c, k, wide, f, inv);
    }
}

// Rows whose codes take stores of VEC bytes.
template <int VEC>
bool wide_codes(const uint8_t* q, uint64_t ld_q) {
    return (uintptr_t)q % VEC == 0 && ld_q % VEC == 0;
}

int check(const char* what, const void* d_x, int dtype, uint32_t rows, uint32_t k, uint64_t ld_x, const uint8_t* d_q,
          uint64_t ld_q, const float* d_scale, uint64_t ld_scale, uint64_t need) {
    if (dtype != LRS_F32 && dtype != LRS_BF16 && dtype != LRS_F16)
        return lrs_call_error(LRS_E_INVALID, "%s: dtype %d", what, dtype);
    if (!d_x || !d_q || !d_scale) return lrs_call_error(LRS_E_INVALID, "%s: NULL buffer", what);
    if (rows > (1u << 24) || k == 0 || k > (1u << 18))
        return lrs_call_error(LRS_E_INVALID, "%s: rows %u / k %u out of range", what, rows, k);
    if (ld_x < k || ld_q < k || ld_scale < need)
        return lrs_call_error(LRS_E_INVALID, "%s: a leading dimension is shorter than its rows", what);
    if ((uintptr_t)d_x % (dtype == LRS_F32 ? 4 : 2) || (uintptr_t)d_scale % 4)
        return lrs_call_error(LRS_E_INVALID, "%s: a buffer is not aligned to its type", what);
    return LRS_OK;
}

template <typename T, int VEC, bool ALIGNED>
int launch_rows(const void* d_x, uint32_t rows, uint32_t k, uint64_t ld_x, uint8_t* d_q, uint64_t ld_q, float* d_scale,
                 uint64_t ld_scale, cudaStream_t s) {
    const uint32_t blocks = (k + kBlock - 1) / kBlock;
    const uint64_t units = (uint64_t)((rows + kRows - 1) / kRows) * blocks, per = kThreads / (kBlock / VEC);
    return launch_kernel("lrs_quantize_rows", quantize_rows_kernel<T, ALIGNED>, (unsigned)((units + per - 1) / per), kThreads, 0, s,
                         static_cast<const T*>(d_x), rows, k, ld_x, d_q, ld_q, d_scale, ld_scale, blocks, wide_codes<VEC>(d_q, ld_q));
}

template <typename T, int VEC, bool ALIGNED>
int launch_blocks(const void* d_x, uint32_t rows, uint32_t k, uint64_t ld_x, uint8_t* d_q, uint64_t ld_q,
                  float* d_scale, uint64_t ld_scale, cudaStream_t s) {
    const uint32_t blocks = (k + kBlock - 1) / kBlock, tall = (rows + kBlock - 1) / kBlock;
    return launch_kernel("lrs_quantize_blocks", quantize_blocks_kernel<T, ALIGNED>, tall * blocks, 16 * sizeof(T) * 8, 0, s,
                         static_cast<const T*>(d_x), rows, k, ld_x, d_q, ld_q, d_scale, ld_scale, blocks, wide_codes<VEC>(d_q, ld_q));
}

template <typename T, int VEC>
int launch_any(bool tall, const void* d_x, uint32_t rows, uint32_t k, uint64_t ld_x, uint8_t* d_q, uint64_t ld_q,
               float* d_scale, uint64_t ld_scale, cudaStream_t s) {
    const bool aligned = (uintptr_t)d_x % 16 == 0 && (rows == 1 || ld_x * sizeof(T) % 16 == 0);
    auto run = tall ? aligned ? launch_blocks<T, VEC, true> : launch_blocks<T, VEC, false>
                    : aligned ? launch_rows<T, VEC, true> : launch_rows<T, VEC, false>;
    return run(d_x, rows, k, ld_x, d_q, ld_q, d_scale, ld_scale, s);
}

}  // namespace

extern "C" int lrs_quantize_rows(const void* d_x, int dtype, uint32_t rows, uint32_t k, uint64_t ld_x, uint8_t* d_q,
                                 uint64_t ld_q, float* d_scale, uint64_t ld_scale, void* stream) {
    if (rows == 0) return LRS_OK;
    const int rc = check("lrs_quantize_rows", d_x, dtype, rows, k, ld_x, d_q, ld_q, d_scale, ld_scale, rows);
    if (rc != LRS_OK) return rc;
    auto run = dtype == LRS_F32 ? launch_any<float, 4> : dtype == LRS_BF16 ? launch_any<__nv_bfloat16, 8> : launch_any<__half, 8>;
    return run(false, d_x, rows, k, ld_x, d_q, ld_q, d_scale, ld_scale, (cudaStream_t)stream);
}

extern "C" int lrs_quantize_blocks(const void* d_x, int dtype, uint32_t rows, uint32_t k, uint64_t ld_x, uint8_t* d_q,
                                   uint64_t ld_q, float* d_scale, uint64_t ld_scale, void* stream) {
    if (rows == 0) return LRS_OK;
    const int rc = check("lrs_quantize_blocks", d_x, dtype, rows, k, ld_x, d_q, ld_q, d_scale, ld_scale,
                         ((uint64_t)k + kBlock - 1) / kBlock);
    if (rc != LRS_OK) return rc;
    auto run = dtype == LRS_F32 ? launch_any<float, 4> : dtype == LRS_BF16 ? launch_any<__nv_bfloat16, 8> : launch_any<__half, 8>;
    return run(true, d_x, rows, k, ld_x, d_q, ld_q, d_scale, ld_scale, (cudaStream_t)stream);
}
