// lrs_head.cu — the language-model head's product in 8-bit floating point (sm_100a):
//   out[r][v] = sum over blocks b of sa[b][r] sw[v / 128][b] (sum over the block of a[r][c] w[v][c])
#include <cuda_fp8.h>

#include "lrs_ops.cuh"

namespace {

using namespace lrs;

constexpr uint32_t kBlock = 128;

// 16 rows x 64 vocabulary entries a CTA, a block of 128 columns at a time in shared memory.
template <typename T>
__global__ void __launch_bounds__(256) head_kernel(const uint8_t* __restrict__ a, uint64_t ld_a,
                                                   const float* __restrict__ sa, uint64_t ld_as,
                                                   const uint8_t* __restrict__ w, uint64_t ld_w,
                                                   const float* __restrict__ sw, uint64_t ld_ws, uint32_t rows,
                                                   uint32_t n, uint32_t k, T* __restrict__ out, uint64_t ld_out) {
    __shared__ float as[16][kBlock + 1], ws[64][kBlock + 1];
    const uint32_t v0 = blockIdx.x * 64, r0 = blockIdx.y * 16;
    const uint32_t tv = threadIdx.x % 64, tr = threadIdx.x / 64;
    float acc[4] = {};
    auto value = [](uint8_t code) {
        __nv_fp8_e4m3 f;
        f.__x = code;
        return (float)f;
    };
    for (uint32_t b = 0; b * kBlock < k; ++b) {
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < 16 * kBlock; i += 256) {
            const uint32_t r = r0 + i / kBlock, c = b * kBlock + i % kBlock;
            as[i / kBlock][i % kBlock] = r < rows && c < k ? value(a[r * ld_a + c]) : 0.0f;
        }
        for (uint32_t i = threadIdx.x; i < 64 * kBlock; i += 256) {
            const uint32_t v = v0 + i / kBlock, c = b * kBlock + i % kBlock;
            ws[i / kBlock][i % kBlock] = v < n && c < k ? value(w[v * ld_w + c]) : 0.0f;
        }
        __syncthreads();
        float s[4] = {};
        for (uint32_t c = 0; c < kBlock; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[j] += as[tr + 4 * j][c] * ws[tv][c];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (r0 + tr + 4 * j < rows && v0 + tv < n)
                acc[j] += s[j] * (sa[b * ld_as + r0 + tr + 4 * j] * sw[(v0 + tv) / kBlock * ld_ws + b]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (r0 + tr + 4 * j < rows && v0 + tv < n) out[(r0 + tr + 4 * j) * ld_out + v0 + tv] = from_float<T>(acc[j]);
}

template <typename T>
int launch(const uint8_t* d_a, uint64_t ld_a, const float* d_as, uint64_t ld_as, const uint8_t* d_w, uint64_t ld_w,
           const float* d_ws, uint64_t ld_ws, uint32_t rows, uint32_t n, uint32_t k, void* d_out, uint64_t ld_out,
           cudaStream_t s) {
    for (uint32_t r = 0; r < rows; r += 16 * 65535) {
        const uint32_t m = rows - r < 16 * 65535 ? rows - r : 16 * 65535;
        head_kernel<T><<<dim3((n + 63) / 64, (m + 15) / 16), 256, 0, s>>>(
            d_a + r * ld_a, ld_a, d_as + r, ld_as, d_w, ld_w, d_ws, ld_ws, m, n, k, (T*)d_out + r * ld_out, ld_out);
    }
    return launched("lrs_fp8_logits");
}

}  // namespace

extern "C" int lrs_fp8_logits(const uint8_t* d_a, uint64_t ld_a, const float* d_a_scale, uint64_t ld_as,
                              const uint8_t* d_w, uint64_t ld_w, const float* d_w_scale, uint64_t ld_ws, uint32_t rows,
                              uint32_t n, uint32_t k, void* d_out, int out_dtype, uint64_t ld_out, void* stream) {
    if (rows == 0) return LRS_OK;
    if (out_dtype != LRS_F32 && out_dtype != LRS_BF16 && out_dtype != LRS_F16)
        return lrs_call_error(LRS_E_INVALID, "lrs_fp8_logits: out_dtype %d", out_dtype);
    if (!d_a || !d_a_scale || !d_w || !d_w_scale || !d_out)
        return lrs_call_error(LRS_E_INVALID, "lrs_fp8_logits: NULL buffer");
    if (rows > (1u << 24) || n == 0 || n > (1u << 24) || k == 0 || k > (1u << 18))
        return lrs_call_error(LRS_E_INVALID, "lrs_fp8_logits: rows %u / n %u / k %u out of range", rows, n, k);
    if (ld_a < k || ld_w < k || ld_as < rows || ld_ws < (k + kBlock - 1) / kBlock || ld_out < n)
        return lrs_call_error(LRS_E_INVALID, "lrs_fp8_logits: a leading dimension is shorter than its rows");
    if ((uintptr_t)d_a % 16 || (uintptr_t)d_w % 16 || (rows > 1 && ld_a % 16) || (n > 1 && ld_w % 16))
        return lrs_call_error(LRS_E_INVALID, "lrs_fp8_logits: codes not on 16-byte boundaries");
    if ((uintptr_t)d_a_scale % 4 || (uintptr_t)d_w_scale % 4 || (uintptr_t)d_out % (out_dtype == LRS_F32 ? 4 : 2))
        return lrs_call_error(LRS_E_INVALID, "lrs_fp8_logits: a buffer is not aligned to its type");
    auto run = out_dtype == LRS_F32 ? launch<float> : out_dtype == LRS_BF16 ? launch<__nv_bfloat16> : launch<__half>;
    return run(d_a, ld_a, d_a_scale, ld_as, d_w, ld_w, d_w_scale, ld_ws, rows, n, k, d_out, ld_out, (cudaStream_t)stream);
}
