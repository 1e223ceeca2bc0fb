// lrs_head.cu — the language-model head's product in 8-bit floating point (sm_100a):
//   out[r][v] = sum over blocks b of sa[b][r] sw[v / 128][b] (sum over the block of a[r][c] w[v][c])
//
// The weights are the tensor core's 128-row operand and the hidden states its other one, so a few
// rows (a decode step) cost a narrow instruction and not a padded one, and a warp's 32 lanes hold 32
// consecutive logits of one row.  A block of 128 columns is one step: four tcgen05.mma (kind
// f8f6f4, K = 32) into TMEM from zero, read back by the epilogue warps and added to f32 registers
// with the block's scale, while the tensor core fills the other TMEM buffer.
//
// Persistent CTAs of twelve warps: 0 issues the TMA copies of both operands (128-byte swizzle, a
// ring of stages), 1 issues the MMAs, 2 brings the scales of a step (4-byte asynchronous copies: any
// alignment), 4-11 are the epilogue, a quarter of the lanes and half of the columns each.  Tiles walk
// the row tiles first, so that the CTAs share the weights they stream in L2.
#include <cuda.h>

#include "lrs_ops.cuh"

namespace {

using namespace lrs;

constexpr uint32_t kBlock = 128;      // columns a scale covers, and columns of a step
constexpr uint32_t kTileV = 128;      // vocabulary entries of a tile
constexpr uint32_t kMaxTileR = 256;   // rows of a tile at most
constexpr uint32_t kThreads = 384;
constexpr uint32_t kEpilogueWarps = 8;
constexpr uint32_t kScaleStages = 8;
constexpr uint32_t kMaxStages = 10;
constexpr long long kWaitCycles = 1ll << 32;  // about 2 s: no wait of a sound launch comes near it

__device__ __forceinline__ uint32_t smem_of(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    return done != 0;
}
// Waits for a phase; false when the bound has passed or another warp has given up.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile uint32_t* lost) {
    if (bar_try(bar, parity)) return true;
    const long long t0 = clock64();
    do {
        if (bar_try(bar, parity)) return true;
        if (*lost) return false;
    } while (clock64() - t0 < kWaitCycles);
    *lost = 1;
    return false;
}

__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, uint32_t x, uint32_t y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}

// K-major operand, 128-byte swizzle: 8 rows of 128 bytes an atom, 1024 bytes from atom to atom.
__device__ __forceinline__ uint64_t operand(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | 1ull << 16 | 64ull << 32 | 1ull << 46 | 2ull << 61;
}
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
        : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void tmem_load(uint32_t addr, float (&v)[8]) {
    uint32_t r[8];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(addr)
                 : "memory");
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_load(uint32_t addr, float (&v)[16]) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
        "[%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

// Completes the loads: the registers pass through, so that nothing reads them earlier.
__device__ __forceinline__ void tmem_wait(float (&v)[8]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7])::"memory");
}
__device__ __forceinline__ void tmem_wait(float (&v)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                   "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15])::"memory");
}

struct Args {
    const float* sa;
    const float* sw;
    void* out;
    uint64_t ld_as, ld_ws, ld_out;
    uint32_t rows, n, blocks;        // blocks of 128 columns
    uint32_t tile_r, row_tiles;      // rows of a tile (16, or a multiple of 32), tiles over the rows
    uint32_t tiles;                  // all of them
    uint32_t stages, tmem_cols;
};

struct Barriers {
    uint64_t full[kMaxStages], empty[kMaxStages];
    uint64_t sfull[kScaleStages], sempty[kScaleStages];
    uint64_t tfull[2], tempty[2];
    uint64_t drain;
    uint32_t tmem;
    uint32_t lost;
};

// HALF: columns of an epilogue warp at most (half of tile_r); CHUNK: columns of one TMEM load.
template <typename T, int HALF, int CHUNK>
__global__ void __launch_bounds__(kThreads, 1) head_kernel(const __grid_constant__ CUtensorMap map_w,
                                                           const __grid_constant__ CUtensorMap map_a, const Args g) {
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ Barriers bars;
    __shared__ __align__(16) float scales[kScaleStages][kMaxTileR + 4];
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t base = (smem_of(smem) + 1023u) & ~1023u;
    const uint32_t stage_bytes = kTileV * kBlock + g.tile_r * kBlock;
    volatile uint32_t* lost = &bars.lost;

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < g.stages; ++s) {
            bar_init(smem_of(&bars.full[s]), 1);
            bar_init(smem_of(&bars.empty[s]), 1);
        }
        for (uint32_t s = 0; s < kScaleStages; ++s) {
            bar_init(smem_of(&bars.sfull[s]), 32);
            bar_init(smem_of(&bars.sempty[s]), kEpilogueWarps);
        }
        for (uint32_t s = 0; s < 2; ++s) {
            bar_init(smem_of(&bars.tfull[s]), 1);
            bar_init(smem_of(&bars.tempty[s]), kEpilogueWarps);
        }
        bar_init(smem_of(&bars.drain), 1);
        bars.lost = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_of(&bars.tmem)),
                     "r"(g.tmem_cols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *(volatile uint32_t*)&bars.tmem;

    if (warp == 0) {
        if (lane == 0) {
            uint32_t it = 0;
            bool ok = true;
            for (uint32_t t = blockIdx.x; ok && t < g.tiles; t += gridDim.x) {
                const uint32_t r0 = t % g.row_tiles * g.tile_r, v0 = t / g.row_tiles * kTileV;
                for (uint32_t b = 0; b < g.blocks; ++b, ++it) {
                    const uint32_t s = it % g.stages;
                    ok = bar_wait(smem_of(&bars.empty[s]), (it / g.stages & 1) ^ 1, lost);
                    if (!ok) break;
                    const uint32_t bar = smem_of(&bars.full[s]), at = base + s * stage_bytes;
                    bar_expect(bar, stage_bytes);
                    tma_load(at, &map_w, b * kBlock, v0, bar);
                    tma_load(at + kTileV * kBlock, &map_a, b * kBlock, r0, bar);
                }
            }
            // (copies that a warp which gave up did not wait for land before the CTA ends)
            if (!ok)
                for (uint32_t j = it > g.stages ? it - g.stages : 0; j < it; ++j) {
                    const long long t0 = clock64();
                    while (!bar_try(smem_of(&bars.full[j % g.stages]), j / g.stages & 1) && clock64() - t0 < kWaitCycles) {
                    }
                }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            const uint32_t idesc = 1u << 4 | g.tile_r / 8 << 17 | kTileV / 16 << 24;  // f32 += e4m3 x e4m3, both K-major
            uint32_t it = 0;
            bool ok = true;
            for (uint32_t t = blockIdx.x; ok && t < g.tiles; t += gridDim.x) {
                for (uint32_t b = 0; b < g.blocks; ++b, ++it) {
                    const uint32_t s = it % g.stages, buf = it & 1;
                    ok = bar_wait(smem_of(&bars.tempty[buf]), (it / 2 & 1) ^ 1, lost) &&
                         bar_wait(smem_of(&bars.full[s]), it / g.stages & 1, lost);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t at = base + s * stage_bytes, d = tmem + buf * (g.tmem_cols / 2);
                    const uint64_t da = operand(at), db = operand(at + kTileV * kBlock);
#pragma unroll
                    for (uint32_t j = 0; j < 4; ++j) mma(d, da + 2 * j, db + 2 * j, idesc, j > 0);
                    mma_commit(smem_of(&bars.empty[s]));
                    mma_commit(smem_of(&bars.tfull[buf]));
                }
            }
            // every MMA has ended before the TMEM goes back
            mma_commit(smem_of(&bars.drain));
            const long long t0 = clock64();
            while (!bar_try(smem_of(&bars.drain), 0) && clock64() - t0 < kWaitCycles) {
            }
        }
        __syncwarp();
    } else if (warp == 2) {
        uint32_t it = 0;
        bool ok = true;
        for (uint32_t t = blockIdx.x; ok && t < g.tiles; t += gridDim.x) {
            const uint32_t r0 = t % g.row_tiles * g.tile_r, v = t / g.row_tiles;
            for (uint32_t b = 0; b < g.blocks; ++b, ++it) {
                const uint32_t s = it % kScaleStages;
                ok = bar_wait(smem_of(&bars.sempty[s]), (it / kScaleStages & 1) ^ 1, lost);
                if (!ok) break;
                const float* src = g.sa + b * g.ld_as + r0;
                for (uint32_t c = lane; c < g.tile_r; c += 32) {
                    const bool in = r0 + c < g.rows;
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_of(&scales[s][c])),
                                 "l"(in ? src + c : g.sa), "r"(in ? 4u : 0u)
                                 : "memory");
                }
                if (lane == 0)
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_of(&scales[s][kMaxTileR])),
                                 "l"(g.sw + v * g.ld_ws + b)
                                 : "memory");
                asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_of(&bars.sfull[s])) : "memory");
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (warp >= 4) {
        const uint32_t e = warp - 4, quarter = e % 4, half = g.tile_r / 2, c0 = e / 4 * half;
        const uint32_t lanes = tmem + (quarter * 32 << 16) + c0;
        uint32_t it = 0;
        bool ok = true;
        for (uint32_t t = blockIdx.x; t < g.tiles; t += gridDim.x) {
            const uint32_t r0 = t % g.row_tiles * g.tile_r + c0, v = t / g.row_tiles * kTileV + quarter * 32 + lane;
            float acc[HALF];
#pragma unroll
            for (int i = 0; i < HALF; ++i) acc[i] = 0.0f;
            for (uint32_t b = 0; ok && b < g.blocks; ++b, ++it) {
                const uint32_t s = it % kScaleStages, buf = it & 1;
                ok = bar_wait(smem_of(&bars.sfull[s]), it / kScaleStages & 1, lost) &&
                     bar_wait(smem_of(&bars.tfull[buf]), it / 2 & 1, lost);
                ok = __all_sync(0xFFFFFFFFu, ok);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const float sw = scales[s][kMaxTileR];
#pragma unroll
                for (int c = 0; c < HALF; c += CHUNK) {
                    if (c < (int)half) {
                        float d[CHUNK];
                        tmem_load(lanes + buf * (g.tmem_cols / 2) + c, d);
                        tmem_wait(d);
#pragma unroll
                        for (int i = 0; i < CHUNK; i += 4) {
                            const float4 sc = *reinterpret_cast<const float4*>(&scales[s][c0 + c + i]);
                            acc[c + i] = fmaf(d[i], sc.x * sw, acc[c + i]);
                            acc[c + i + 1] = fmaf(d[i + 1], sc.y * sw, acc[c + i + 1]);
                            acc[c + i + 2] = fmaf(d[i + 2], sc.z * sw, acc[c + i + 2]);
                            acc[c + i + 3] = fmaf(d[i + 3], sc.w * sw, acc[c + i + 3]);
                        }
                    }
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    bar_arrive(smem_of(&bars.tempty[buf]));
                    bar_arrive(smem_of(&bars.sempty[s]));
                }
            }
            // (a wait that ran out leaves NaN, which the samplers report)
            T* out = reinterpret_cast<T*>(g.out) + (uint64_t)r0 * g.ld_out + v;
#pragma unroll
            for (int i = 0; i < HALF; ++i)
                if (i < (int)half && r0 + i < g.rows && v < g.n)
                    out[i * g.ld_out] = from_float<T>(ok ? acc[i] : __int_as_float(0x7FC00000));
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1) {
        __syncwarp();
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(g.tmem_cols) : "memory");
    }
}

typedef CUresult (*encode_t)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                             const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

encode_t encoder() {
    static const encode_t f = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult st;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &st) != cudaSuccess ||
            st != cudaDriverEntryPointSuccess)
            p = nullptr;
        return (encode_t)p;
    }();
    return f;
}

// rows x k codes, read in boxes of 128 columns x `box` rows (zeros outside).
bool code_map(CUtensorMap* m, const uint8_t* p, uint32_t rows, uint32_t k, uint64_t ld, uint32_t box) {
    const cuuint64_t dims[2] = {k, rows};
    const cuuint64_t strides[1] = {rows > 1 ? ld : ((uint64_t)k + 15) / 16 * 16};
    const cuuint32_t boxes[2] = {kBlock, box}, step[2] = {1, 1};
    return encoder()(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(p), dims, strides, boxes, step,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct DeviceInfo {
    int sms = 0, smem = 0;
};

constexpr int kMaxDevices = 64;

template <typename T, int HALF, int CHUNK>
int launch(const CUtensorMap& mw, const CUtensorMap& ma, Args g, cudaStream_t s) {
    int dev = 0;
    static DeviceInfo info[kMaxDevices];  // (every thread that fills an entry writes the same values)
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices)
        return lrs_call_error(LRS_E_CUDA, "lrs_fp8_logits: no current device");
    auto* kernel = head_kernel<T, HALF, CHUNK>;
    if (info[dev].sms == 0) {
        int sms = 0, smem = 0;
        cudaFuncAttributes at;
        cudaError_t e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
        if (e == cudaSuccess) e = cudaDeviceGetAttribute(&smem, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev);
        if (e == cudaSuccess) e = cudaFuncGetAttributes(&at, kernel);
        if (e == cudaSuccess) smem -= (int)at.sharedSizeBytes;
        if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return lrs_call_error(LRS_E_CUDA, "lrs_fp8_logits: %s", cudaGetErrorString(e));
        info[dev].smem = smem;
        info[dev].sms = sms;
    }
    const uint32_t stage = (kTileV + g.tile_r) * kBlock;
    g.stages = ((uint32_t)info[dev].smem - 1024) / stage;
    if (g.stages > kMaxStages) g.stages = kMaxStages;
    const uint32_t grid = g.tiles < (uint32_t)info[dev].sms ? g.tiles : (uint32_t)info[dev].sms;
    kernel<<<grid, kThreads, g.stages * stage + 1024, s>>>(mw, ma, g);
    return launched("lrs_fp8_logits");
}

template <typename T>
int run(const CUtensorMap& mw, const CUtensorMap& ma, const Args& g, cudaStream_t s) {
    if (g.tile_r == 16) return launch<T, 8, 8>(mw, ma, g, s);
    if (g.tile_r <= 64) return launch<T, 32, 16>(mw, ma, g, s);
    if (g.tile_r <= 128) return launch<T, 64, 16>(mw, ma, g, s);
    return launch<T, 128, 16>(mw, ma, g, s);
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
    if (!encoder()) return lrs_call_error(LRS_E_CUDA, "lrs_fp8_logits: the driver has no cuTensorMapEncodeTiled");
    Args g{};
    g.sa = d_a_scale, g.sw = d_w_scale, g.out = d_out;
    g.ld_as = ld_as, g.ld_ws = ld_ws, g.ld_out = ld_out;
    g.rows = rows, g.n = n, g.blocks = (k + kBlock - 1) / kBlock;
    // the fewest row tiles of at most 256 rows, of equal size in the tensor core's steps
    g.row_tiles = (rows + kMaxTileR - 1) / kMaxTileR;
    const uint32_t each = (rows + g.row_tiles - 1) / g.row_tiles;
    g.tile_r = each <= 16 ? 16 : (each + 31) / 32 * 32;
    g.row_tiles = (rows + g.tile_r - 1) / g.tile_r;
    const uint64_t tiles = (uint64_t)g.row_tiles * ((n + kTileV - 1) / kTileV);
    if (tiles > 0x7FFFFFFFu) return lrs_call_error(LRS_E_INVALID, "lrs_fp8_logits: rows x n too large");
    g.tiles = (uint32_t)tiles;
    g.tmem_cols = 32;
    while (g.tmem_cols < 2 * g.tile_r) g.tmem_cols *= 2;
    CUtensorMap mw, ma;
    if (!code_map(&mw, d_w, n, k, ld_w, kTileV) || !code_map(&ma, d_a, rows, k, ld_a, g.tile_r))
        return lrs_call_error(LRS_E_INVALID, "lrs_fp8_logits: the codes cannot be mapped (ld too large?)");
    const cudaStream_t s = (cudaStream_t)stream;
    return out_dtype == LRS_F32 ? run<float>(mw, ma, g, s) : out_dtype == LRS_BF16 ? run<__nv_bfloat16>(mw, ma, g, s) : run<__half>(mw, ma, g, s);
}
