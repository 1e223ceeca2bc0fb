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

// VEC elements of a row from column c on, zeros past k; one 16-byte load where `wide` (16-byte
// aligned rows) and the elements are all there.
template <typename T, int VEC>
__device__ __forceinline__ void load(const T* row, uint32_t c, uint32_t k, bool wide, float (&x)[VEC]) {
    if (wide && c + VEC <= k) {
        unpack(*reinterpret_cast<const uint4*>(row + c), x, row);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) x[i] = c + i < k ? to_float<T>(row[c + i]) : 0.0f;
    }
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

template <int VEC>
__device__ __forceinline__ float amax(const float (&x)[VEC], float m) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) m = max_nan(m, fabsf(x[i]));
    return m;
}

// A group of 128 / VEC lanes takes one block of 128 columns of kRows consecutive rows: kRows
// loads in flight a lane, and the block's kRows scales (block-major) go out in one store each of
// consecutive lanes.
constexpr int kRows = 8;

template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const T* __restrict__ x, uint32_t rows, uint32_t k,
                                                                 uint64_t ld_x, uint8_t* __restrict__ q, uint64_t ld_q,
                                                                 float* __restrict__ scale, uint64_t ld_scale,
                                                                 uint32_t blocks, bool wide) {
    constexpr uint32_t kLanes = kBlock / VEC;
    const uint64_t unit = ((uint64_t)blockIdx.x * kThreads + threadIdx.x) / kLanes;
    const uint32_t lane = threadIdx.x % kLanes;
    const uint32_t b = (uint32_t)(unit % blocks);
    const uint64_t r0 = unit / blocks * kRows;
    if (r0 >= rows) return;  // (whole groups leave: the shuffles below stay within a group)
    const uint32_t c = b * kBlock + lane * VEC;
    float v[kRows][VEC], s[kRows];
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
        if (r0 + j < rows) {
            load<T, VEC>(x + (r0 + j) * ld_x, c, k, wide, v[j]);
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[j][i] = 0.0f;
        }
    }
    const uint32_t mask = kLanes == 32 ? 0xFFFFFFFFu : 0xFFFFu << (threadIdx.x & 16u);
    float mine = 0.0f;
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
        float m = amax(v[j], 0.0f);
#pragma unroll
        for (uint32_t o = kLanes / 2; o > 0; o /= 2) m = max_nan(m, __shfl_xor_sync(mask, m, o));
        s[j] = scale_of(m);
        if (lane == j) mine = s[j];
    }
    if (lane < kRows && r0 + lane < rows) scale[b * ld_scale + r0 + lane] = mine;
#pragma unroll
    for (int j = 0; j < kRows; ++j)
        if (r0 + j < rows) store<VEC>(q + (r0 + j) * ld_q, c, k, wide, v[j], __frcp_rn(s[j]));
}

// One CTA takes one 128 x 128 block, 64 elements a thread.
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) quantize_blocks_kernel(const T* __restrict__ x, uint32_t rows, uint32_t k,
                                                                   uint64_t ld_x, uint8_t* __restrict__ q, uint64_t ld_q,
                                                                   float* __restrict__ scale, uint64_t ld_scale,
                                                                   uint32_t blocks, bool wide) {
    constexpr uint32_t kLanes = kBlock / VEC, kStep = kThreads / kLanes;
    constexpr int kN = kBlock / kStep;
    __shared__ float part[kThreads / 32];
    const uint32_t a = blockIdx.x / blocks, b = blockIdx.x % blocks;
    const uint32_t c = b * kBlock + threadIdx.x % kLanes * VEC;
    const uint64_t r0 = (uint64_t)a * kBlock + threadIdx.x / kLanes;
    float v[kN][VEC], m = 0.0f;
#pragma unroll
    for (int j = 0; j < kN; ++j) {
        const uint64_t r = r0 + j * kStep;
        if (r < rows) {
            load<T, VEC>(x + r * ld_x, c, k, wide, v[j]);
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[j][i] = 0.0f;
        }
    }
#pragma unroll
    for (int j = 0; j < kN; ++j) m = amax(v[j], m);
#pragma unroll
    for (uint32_t o = 16; o > 0; o /= 2) m = max_nan(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = m;
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < kThreads / 32; ++w) m = max_nan(m, part[w]);
    const float s = scale_of(m), inv = __frcp_rn(s);
    if (threadIdx.x == 0) scale[a * ld_scale + b] = s;
#pragma unroll
    for (int j = 0; j < kN; ++j) {
        const uint64_t r = r0 + j * kStep;
        if (r < rows) store<VEC>(q + r * ld_q, c, k, wide, v[j], inv);
    }
}

// Rows that take 16-byte loads and VEC-byte stores.
template <int VEC>
bool wide_rows(const void* x, uint64_t ld_x, size_t size, const uint8_t* q, uint64_t ld_q) {
    return (uintptr_t)x % 16 == 0 && ld_x * size % 16 == 0 && (uintptr_t)q % VEC == 0 && ld_q % VEC == 0;
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

template <typename T, int VEC>
void launch_rows(const void* d_x, uint32_t rows, uint32_t k, uint64_t ld_x, uint8_t* d_q, uint64_t ld_q, float* d_scale,
                 uint64_t ld_scale, cudaStream_t s) {
    const uint32_t blocks = (k + kBlock - 1) / kBlock;
    const uint64_t units = (uint64_t)((rows + kRows - 1) / kRows) * blocks, per = kThreads / (kBlock / VEC);
    quantize_rows_kernel<T, VEC><<<(unsigned)((units + per - 1) / per), kThreads, 0, s>>>(
        (const T*)d_x, rows, k, ld_x, d_q, ld_q, d_scale, ld_scale, blocks, wide_rows<VEC>(d_x, ld_x, sizeof(T), d_q, ld_q));
}

template <typename T, int VEC>
void launch_blocks(const void* d_x, uint32_t rows, uint32_t k, uint64_t ld_x, uint8_t* d_q, uint64_t ld_q,
                   float* d_scale, uint64_t ld_scale, cudaStream_t s) {
    const uint32_t blocks = (k + kBlock - 1) / kBlock, tall = (rows + kBlock - 1) / kBlock;
    quantize_blocks_kernel<T, VEC><<<tall * blocks, kThreads, 0, s>>>(
        (const T*)d_x, rows, k, ld_x, d_q, ld_q, d_scale, ld_scale, blocks, wide_rows<VEC>(d_x, ld_x, sizeof(T), d_q, ld_q));
}

}  // namespace

extern "C" int lrs_quantize_rows(const void* d_x, int dtype, uint32_t rows, uint32_t k, uint64_t ld_x, uint8_t* d_q,
                                 uint64_t ld_q, float* d_scale, uint64_t ld_scale, void* stream) {
    if (rows == 0) return LRS_OK;
    const int rc = check("lrs_quantize_rows", d_x, dtype, rows, k, ld_x, d_q, ld_q, d_scale, ld_scale, rows);
    if (rc != LRS_OK) return rc;
    auto run = dtype == LRS_F32 ? launch_rows<float, 4> : dtype == LRS_BF16 ? launch_rows<__nv_bfloat16, 8> : launch_rows<__half, 8>;
    run(d_x, rows, k, ld_x, d_q, ld_q, d_scale, ld_scale, (cudaStream_t)stream);
    return launched("lrs_quantize_rows");
}

extern "C" int lrs_quantize_blocks(const void* d_x, int dtype, uint32_t rows, uint32_t k, uint64_t ld_x, uint8_t* d_q,
                                   uint64_t ld_q, float* d_scale, uint64_t ld_scale, void* stream) {
    if (rows == 0) return LRS_OK;
    const int rc = check("lrs_quantize_blocks", d_x, dtype, rows, k, ld_x, d_q, ld_q, d_scale, ld_scale,
                         ((uint64_t)k + kBlock - 1) / kBlock);
    if (rc != LRS_OK) return rc;
    auto run = dtype == LRS_F32 ? launch_blocks<float, 4> : dtype == LRS_BF16 ? launch_blocks<__nv_bfloat16, 8> : launch_blocks<__half, 8>;
    run(d_x, rows, k, ld_x, d_q, ld_q, d_scale, ld_scale, (cudaStream_t)stream);
    return launched("lrs_quantize_blocks");
}
