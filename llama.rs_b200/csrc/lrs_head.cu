// lrs_head.cu — the language-model head's product in 8-bit floating point (sm_100a):
//   out[r][v] = sum over blocks b of sa[b][r] sw[v / 128][b] (sum over the block of a[r][c] w[v][c])
//
// A block of 128 columns is one step: four tcgen05.mma (kind f8f6f4, K = 32) into TMEM from zero, read
// back by the epilogue warps and added to f32 registers with the block's scales, while the tensor core
// fills another TMEM buffer.  Persistent CTAs: warp 0 issues the TMA copies of both operands
// (128-byte swizzle, a ring of stages), 1 issues the MMAs, the last 16 are the epilogue.  Tiles walk the row
// tiles first, so that the CTAs share the weights they stream in L2.  Two forms:
//   narrow  up to 32 or 64 rows (a decode step; bound by the weights' bytes): the weights are the tensor core's
//           128-row operand, so a few rows cost a narrow instruction and not a padded one, and a warp's
//           lanes are consecutive logits of one row.  A row is a TMEM column there, its scale the same
//           for a whole warp: warp 2 brings them to shared memory (4-byte asynchronous copies: any
//           alignment), from where a thread reads one for each of its 16 columns.
//   wide    more rows: 128 rows x 256 vocabulary entries.  A row is a TMEM lane, so a thread has one
//           row scale and one weight scale a step and adds with a single factor (with the rows as
//           columns the scales' shared-memory reads and products took three times the MMAs' time); the
//           logits go out through shared memory, 64 bytes of a row at a time.
// Measured (one B200): 1 x 151,936 x 1,024 in 31.8 us (5.0 TB/s); n = 109,051, k = 2,048, bf16 over changing inputs: 1 to 32
// rows in 45 to 47 us (4.9 to 5.0 TB/s, three quarters of the copy rate: the weights' way in), 64 rows in 51 to 59 us (4.0 to
// 4.7), where the epilogue's reads of TMEM and the activations' codes, fetched again for every tile, add to it; 256 x
// 151,936 x 4,096 f32 in 200 us and 1,024 rows in 650 to 680 us (1.9 PFLOP/s; 781 under the power cap), bound by the block
// sums' way through the epilogue warps (tensor pipe 48 % busy).  Rows on no 16-byte boundary cost the wide form a third
// (237 x 109,051 x 1,000: f32 72 us and not 54, bf16 63 and not 47).
#include <cuda.h>

#include <atomic>

#include "lrs_ops.cuh"

namespace {

using namespace lrs;

constexpr uint32_t kBlock = 128;      // columns a scale covers, and columns of a step
// Rows of the narrow form at most, and where rows of d_out start on 16-byte boundaries (the wide form stores others element by
// element).  Measured, narrow and wide, us (one B200): 151,936 x 4,096 bf16 17 rows 108.7 and 134.0, 32 rows 109.6 and 111.3,
// 48 rows 135.5 and 113.4, 64 rows 138.6 and 115.7, 65 rows (two narrow tiles) 258 and 113; 151,936 x 1,024 f32 32 rows 33.9 and 38.0, 64
// rows 40.3 and 41.1, 65 rows 72.0 and 41.2; 32,000 x 2,048 f32 32 rows 16.1 and 15.5, 64 rows 20.1 and 13.6.  Unaligned, 109,051 x
// 2,048 bf16: 32 rows 43.4 and 55.1, 64 rows 50.6 and 52.5, 65 rows 96.2 and 52.7.
constexpr uint32_t kNarrowRows = 64, kNarrowAligned = 32;
constexpr uint32_t kThreads = 640;  // of both forms
constexpr uint32_t kMaxBuffers = 8;   // TMEM accumulators
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
// Position in a ring of barriers.
struct Ring {
    uint32_t at = 0, turn = 0;
    __device__ __forceinline__ void next(uint32_t size) {
        if (++at == size) at = 0, turn ^= 1;
    }
};

__device__ __forceinline__ bool elect() {
    uint32_t one;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(one));
    return one != 0;
}

// Waits for a phase; false when the bound has passed or another warp has given up.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, long long bound, volatile uint32_t* lost) {
    if (bar_try(bar, parity)) return true;
    const long long t0 = clock64();
    do {
        if (bar_try(bar, parity)) return true;
        if (*lost) return false;
    } while (clock64() - t0 < bound);
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

__device__ __forceinline__ void tmem_load(uint32_t addr, float (&v)[32]) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_wait(float (&v)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]), "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]), "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]), "+f"(v[30]), "+f"(v[31]) :: "memory");
}
// Completes the loads: the registers pass through, so that nothing reads them earlier.
__device__ __forceinline__ void tmem_wait(float (&v)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                   "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15])::"memory");
}
__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

struct Args {
    const float* sa;
    const float* sw;
    void* out;
    uint64_t ld_as, ld_ws, ld_out;
    uint32_t rows, n, blocks;          // blocks of 128 columns
    uint32_t tile_r, tile_v;           // rows and vocabulary entries of a tile
    uint32_t row_tiles, tiles;         // tiles over the rows, all of them
    uint32_t first_bytes, stage_bytes; // of the 128-row operand, of a stage
    uint32_t stages, buffers;          // of shared memory, of TMEM
    uint32_t columns, tmem_columns;    // of a buffer, allocated
    bool wide_out;                     // rows of d_out start on 16-byte boundaries
    long long bound;                   // cycles that a wait takes at most
    uint32_t copies;                   // steps that a CTA issues the copies of (all, but in the test of the waits)
};

struct Barriers {
    uint64_t full[kMaxStages], empty[kMaxStages];
    uint64_t sfull[kScaleStages], sempty[kScaleStages];
    uint64_t tfull[kMaxBuffers], tempty[kMaxBuffers];
    uint64_t drain;
    uint32_t tmem;
    uint32_t lost;
};

// Barriers and TMEM of a CTA; `releases` arrivals free a TMEM buffer (and a stage of scales).
__device__ __forceinline__ uint32_t set_up(const Args& g, Barriers& bars, uint32_t releases) {
    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < g.stages; ++s) {
            bar_init(smem_of(&bars.full[s]), 1);
            bar_init(smem_of(&bars.empty[s]), 1);
        }
        for (uint32_t s = 0; s < kScaleStages; ++s) {
            bar_init(smem_of(&bars.sfull[s]), 32);
            bar_init(smem_of(&bars.sempty[s]), releases);
        }
        for (uint32_t s = 0; s < g.buffers; ++s) {
            bar_init(smem_of(&bars.tfull[s]), 1);
            bar_init(smem_of(&bars.tempty[s]), releases);
        }
        bar_init(smem_of(&bars.drain), 1);
        bars.lost = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (threadIdx.x / 32 == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_of(&bars.tmem)),
                     "r"(g.tmem_columns)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    return *(volatile uint32_t*)&bars.tmem;
}

__device__ __forceinline__ void tear_down(const Args& g, uint32_t tmem) {
    tmem_fence_before();
    __syncthreads();
    if (threadIdx.x / 32 == 1) {
        __syncwarp();
        tmem_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(g.tmem_columns) : "memory");
    }
}

// One warp, so that the operands of what its elected lane issues are uniform (as a single thread's they took
// 800 cycles a step and not 300): the copies of both operands of every step, the 128-row one first.
__device__ __forceinline__ void copy_warp(const Args& g, Barriers& bars, uint32_t base, const CUtensorMap* first,
                                            const CUtensorMap* second, bool weights_first) {
    volatile uint32_t* lost = &bars.lost;
    const uint32_t full = smem_of(bars.full), empty = smem_of(bars.empty);
    const bool leader = elect();
    Ring ring;
    uint32_t at = base, issued = 0;
    bool ok = true;
    for (uint32_t t = blockIdx.x; ok && t < g.tiles; t += gridDim.x) {
        const uint32_t r0 = t % g.row_tiles * g.tile_r, v0 = t / g.row_tiles * g.tile_v;
        const uint32_t y0 = weights_first ? v0 : r0, y1 = weights_first ? r0 : v0;
        for (uint32_t b = 0; b < g.blocks; ++b, ++issued) {
            ok = bar_wait(empty + ring.at * 8, ring.turn ^ 1, g.bound, lost);
            if (!ok) break;
            const uint32_t bar = full + ring.at * 8;
            if (leader && issued < g.copies) {
                bar_expect(bar, g.stage_bytes);
                tma_load(at, first, b * kBlock, y0, bar);
                tma_load(at + g.first_bytes, second, b * kBlock, y1, bar);
            }
            ring.next(g.stages);
            at = ring.at == 0 ? base : at + g.stage_bytes;
        }
    }
    // every copy lands before the CTA ends, also where a warp that gave up did not wait for it (the lane that issued
    // them counts them; before a stage's last copy came its `empty`, hence the ones before have landed)
    if (leader) {
        issued = min(issued, g.copies);
        for (uint32_t j = issued > g.stages ? issued - g.stages : 0; j < issued; ++j) {
            const long long t0 = clock64();
            while (!bar_try(full + j % g.stages * 8, j / g.stages & 1) && clock64() - t0 < kWaitCycles) {
            }
        }
    }
}

// One warp: the MMAs of every step, 128 x `columns` into the next TMEM buffer.
__device__ __forceinline__ void mma_warp(const Args& g, Barriers& bars, uint32_t base, uint32_t tmem) {
    volatile uint32_t* lost = &bars.lost;
    const uint32_t idesc = 1u << 4 | g.columns / 8 << 17 | 128 / 16 << 24;  // f32 += e4m3 x e4m3, both K-major
    const uint32_t full = smem_of(bars.full), empty = smem_of(bars.empty), tfull = smem_of(bars.tfull), tempty = smem_of(bars.tempty);
    const uint64_t first = operand(base), second = operand(base + g.first_bytes), step = g.stage_bytes >> 4;
    const bool leader = elect();
    Ring ring, buffer;
    uint64_t da = first, db = second;
    uint32_t d = tmem;
    bool ok = true;
    for (uint32_t t = blockIdx.x; ok && t < g.tiles; t += gridDim.x) {
        for (uint32_t b = 0; b < g.blocks; ++b) {
            ok = bar_wait(tempty + buffer.at * 8, buffer.turn ^ 1, g.bound, lost) &&
                 bar_wait(full + ring.at * 8, ring.turn, g.bound, lost);
            if (!ok) break;
            tmem_fence_after();
            if (leader) {
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) mma(d, da + 2 * j, db + 2 * j, idesc, j > 0);
                mma_commit(empty + ring.at * 8);
                mma_commit(tfull + buffer.at * 8);
            }
            ring.next(g.stages);
            buffer.next(g.buffers);
            da = ring.at == 0 ? first : da + step, db = ring.at == 0 ? second : db + step;
            d = buffer.at == 0 ? tmem : d + g.columns;
        }
    }
    // every MMA has ended before the TMEM goes back
    if (leader) mma_commit(smem_of(&bars.drain));
    const long long t0 = clock64();
    while (!bar_try(smem_of(&bars.drain), 0) && clock64() - t0 < kWaitCycles) {
    }
}

constexpr float kLost = __builtin_nanf("");  // what a wait that ran out leaves: the samplers report it

template <typename T>
__global__ void __launch_bounds__(kThreads, 1) narrow_kernel(const __grid_constant__ CUtensorMap map_w,
                                                             const __grid_constant__ CUtensorMap map_a, const Args g) {
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ Barriers bars;
    __shared__ __align__(16) float scales[kScaleStages][kNarrowRows + 4];
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, groups = g.tile_r / 16;
    const uint32_t base = (smem_of(smem) + 1023u) & ~1023u;
    volatile uint32_t* lost = &bars.lost;
    const uint32_t tmem = set_up(g, bars, 4 * groups);

    if (warp == 0) {
        copy_warp(g, bars, base, &map_w, &map_a, true);
    } else if (warp == 1) {
        mma_warp(g, bars, base, tmem);
    } else if (warp == 2) {
        Ring ring;
        bool ok = true;
        for (uint32_t t = blockIdx.x; ok && t < g.tiles; t += gridDim.x) {
            const uint32_t r0 = t % g.row_tiles * g.tile_r, v = t / g.row_tiles;
            for (uint32_t b = 0; b < g.blocks; ++b) {
                ok = bar_wait(smem_of(&bars.sempty[ring.at]), ring.turn ^ 1, g.bound, lost);
                if (!ok) break;  // (a lane that gives up sends nothing more: the others run out as well)
                const float* src = g.sa + b * g.ld_as + r0;
                for (uint32_t c = lane; c < g.tile_r; c += 32) {
                    const bool in = r0 + c < g.rows;
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_of(&scales[ring.at][c])),
                                 "l"(in ? src + c : g.sa), "r"(in ? 4u : 0u)
                                 : "memory");
                }
                if (lane == 0)
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_of(&scales[ring.at][kNarrowRows])),
                                 "l"(g.sw + v * g.ld_ws + b)
                                 : "memory");
                asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_of(&bars.sfull[ring.at]))
                             : "memory");
                ring.next(kScaleStages);
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (warp >= 4 && warp < 4 + 4 * groups) {
        const uint32_t e = warp - 4, quarter = e % 4, c0 = e / 4 * 16;
        const uint32_t lanes = tmem + (quarter * 32 << 16) + c0;
        Ring ring, buffer;
        bool ok = true;
        for (uint32_t t = blockIdx.x; t < g.tiles; t += gridDim.x) {
            const uint32_t r0 = t % g.row_tiles * g.tile_r + c0, v = t / g.row_tiles * g.tile_v + quarter * 32 + lane;
            float acc[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[i] = 0.0f;
            // (after a wait that ran out the steps go on without waiting, and the tile is lost)
            for (uint32_t b = 0; b < g.blocks; ++b) {
                ok &= bar_wait(smem_of(&bars.sfull[ring.at]), ring.turn, g.bound, lost);
                ok &= bar_wait(smem_of(&bars.tfull[buffer.at]), buffer.turn, g.bound, lost);
                __syncwarp();
                tmem_fence_after();
                float d[16];
                tmem_load(lanes + buffer.at * g.columns, d);
                const float sw = scales[ring.at][kNarrowRows];
                float s[16];
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    const float4 f = *reinterpret_cast<const float4*>(&scales[ring.at][c0 + i]);
                    s[i] = f.x * sw, s[i + 1] = f.y * sw, s[i + 2] = f.z * sw, s[i + 3] = f.w * sw;
                }
                tmem_wait(d);
                tmem_fence_before();
                __syncwarp();
                if (lane == 0) {
                    bar_arrive(smem_of(&bars.tempty[buffer.at]));
                    bar_arrive(smem_of(&bars.sempty[ring.at]));
                }
                ring.next(kScaleStages);
                buffer.next(g.buffers);
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[i] = fmaf(d[i], s[i], acc[i]);
            }
            ok &= *lost == 0;  // (what ran on without waiting may have freed this warp's buffers early)
            T* out = reinterpret_cast<T*>(g.out) + (uint64_t)r0 * g.ld_out + v;
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (r0 + i < g.rows && v < g.n) out[i * g.ld_out] = from_float<T>(ok ? acc[i] : kLost);
        }
    }
    tear_down(g, tmem);
}

// acc += d * s, two columns an instruction
template <int N>
__device__ __forceinline__ void add_scaled(float* acc, const float (&d)[N], float s) {
    const float2 f = make_float2(s, s);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const float2 x = __ffma2_rn(make_float2(d[i], d[i + 1]), f, make_float2(acc[i], acc[i + 1]));
        acc[i] = x.x, acc[i + 1] = x.y;
    }
}

constexpr uint32_t kWideR = 128, kWideV = 256, kWideWarps = 16;
constexpr uint32_t kWideCols = kWideV / (kWideWarps / 4);   // of an epilogue warp
constexpr uint32_t kFewRegs = 32, kManyRegs = 112;          // of the first four warps, of the epilogue's
constexpr uint32_t kWideRegs = 128 * kFewRegs + 512 * kManyRegs;
constexpr uint32_t kPiece = 64;                             // bytes of a row that go out together

template <typename T>
__global__ void __launch_bounds__(kThreads, 1) wide_kernel(const __grid_constant__ CUtensorMap map_a,
                                                           const __grid_constant__ CUtensorMap map_w, const Args g) {
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ Barriers bars;
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t base = (smem_of(smem) + 1023u) & ~1023u;
    volatile uint32_t* lost = &bars.lost;
    const uint32_t tmem = set_up(g, bars, kWideWarps);
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewRegs));
        if (warp == 0) copy_warp(g, bars, base, &map_a, &map_w, false);
        if (warp == 1) mma_warp(g, bars, base, tmem);
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kManyRegs));
        const uint32_t e = warp - 4, quarter = warp % 4, c0 = e / 4 * kWideCols;
        const uint32_t lanes = tmem + (quarter * 32 << 16) + c0;
        const uint32_t tfull = smem_of(bars.tfull), tempty = smem_of(bars.tempty);
        uint8_t* piece = smem + (base - smem_of(smem)) + g.stages * g.stage_bytes + e * 32 * kPiece;
        uint32_t buffer = 0, turn = 0;
        bool ok = true;
        for (uint32_t t = blockIdx.x; t < g.tiles; t += gridDim.x) {
            const uint32_t r0 = t % g.row_tiles * kWideR + quarter * 32, v0 = t / g.row_tiles * kWideV + c0;
            // the scales of this thread's row and of its columns' weights, two steps ahead of their use
            const float* sa = g.sa + min(r0 + lane, g.rows - 1);
            const float* sw = g.sw + min(v0, g.n - 1) / kBlock * g.ld_ws;
            float a0 = __ldg(sa), w0 = __ldg(sw), a1 = a0, w1 = w0;
            if (g.blocks > 1) sa += g.ld_as, ++sw, a1 = __ldg(sa), w1 = __ldg(sw);
            float acc[kWideCols];
#pragma unroll
            for (int i = 0; i < (int)kWideCols; ++i) acc[i] = 0.0f;
            // (after a wait that ran out the steps go on without waiting, and the tile is lost)
            for (uint32_t b = 0; b < g.blocks; ++b) {
                const float s0 = a0 * w0;
                a0 = a1, w0 = w1;
                if (b + 2 < g.blocks) sa += g.ld_as, ++sw, a1 = __ldg(sa), w1 = __ldg(sw);
                ok &= bar_wait(tfull + buffer * 8, turn, g.bound, lost);
                __syncwarp();
                tmem_fence_after();
                const uint32_t from = lanes + buffer * kWideV;
#pragma unroll
                for (int c = 0; c < (int)kWideCols; c += 32) {
                    float d[32];
                    tmem_load(from + c, d);
                    tmem_wait(d);
                    if (c + 32 == (int)kWideCols) {
                        tmem_fence_before();
                        __syncwarp();
                        if (lane == 0) bar_arrive(tempty + buffer * 8);
                    }
                    add_scaled<32>(acc + c, d, s0);
                }
                buffer ^= 1;
                turn ^= buffer == 0;
            }
            ok &= *lost == 0;  // (what ran on without waiting may have freed this warp's buffers early)
            if (!ok) {
#pragma unroll
                for (int i = 0; i < (int)kWideCols; ++i) acc[i] = kLost;
            }
            // a piece of each of the 32 rows through shared memory: a lane writes its row's 16-byte parts,
            // turned by the row so that eight rows meet all banks, and lanes read along the rows
            constexpr uint32_t kCols = kPiece / sizeof(T), kEach = 16 / sizeof(T);
            T* out = reinterpret_cast<T*>(g.out) + (uint64_t)r0 * g.ld_out + v0;
            const uint32_t left = r0 < g.rows ? g.rows - r0 : 0;  // rows of this warp's 32
#pragma unroll
            for (int c = 0; c < (int)kWideCols; c += kCols) {
                __syncwarp();
#pragma unroll
                for (uint32_t q = 0; q < 4; ++q) {
                    uint32_t w[4];
#pragma unroll
                    for (uint32_t i = 0; i < 4; ++i) {
                        if constexpr (sizeof(T) == 4) {
                            w[i] = __float_as_uint(acc[c + q * 4 + i]);
                        } else {
                            const T lo = from_float<T>(acc[c + q * 8 + 2 * i]), hi = from_float<T>(acc[c + q * 8 + 2 * i + 1]);
                            w[i] = (uint32_t) * reinterpret_cast<const uint16_t*>(&lo) |
                                   (uint32_t) * reinterpret_cast<const uint16_t*>(&hi) << 16;
                        }
                    }
                    *reinterpret_cast<uint4*>(piece + lane * kPiece + (q ^ (lane >> 1 & 3)) * 16) = make_uint4(w[0], w[1], w[2], w[3]);
                }
                __syncwarp();
                if (g.wide_out && v0 + c + kCols <= g.n) {  // 16 bytes a lane, eight rows an instruction
                    const uint32_t row0 = lane / 4, part = lane % 4;
                    T* to = out + row0 * g.ld_out + c + part * kEach;
#pragma unroll
                    for (uint32_t row = row0; row < 32; row += 8, to += 8 * g.ld_out) {
                        const uint4 x = *reinterpret_cast<const uint4*>(piece + row * kPiece + (part ^ (row >> 1 & 3)) * 16);
                        if (row < left) *reinterpret_cast<uint4*>(to) = x;
                    }
                } else {
                    constexpr uint32_t kRows = 32 / kCols;  // rows an instruction
                    const uint32_t row0 = lane / kCols, col = lane % kCols, part = col / kEach;
                    const uint32_t end = v0 + c + col < g.n ? left : 0;
                    T* to = out + row0 * g.ld_out + c + col;
#pragma unroll 8
                    for (uint32_t row = row0; row < 32; row += kRows, to += kRows * g.ld_out) {
                        const T x = *reinterpret_cast<const T*>(piece + row * kPiece + (part ^ (row >> 1 & 3)) * 16 + col * sizeof(T) % 16);
                        if (row < end) *to = x;
                    }
                }
            }
        }
    }
    tear_down(g, tmem);
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
    std::atomic<int> sms{0}, smem{0};  // (sms last: it says that both are there)
};

constexpr int kMaxDevices = 64;

template <typename T>
int launch(void (*kernel)(CUtensorMap, CUtensorMap, Args), DeviceInfo* info, const CUtensorMap& first,
           const CUtensorMap& second, Args g, uint32_t regs, uint32_t more, cudaStream_t s) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices)
        return lrs_call_error(LRS_E_CUDA, "lrs_fp8_logits: no current device");
    if (info[dev].sms == 0) {  // (every thread that fills an entry writes the same values)
        int sms = 0, smem = 0;
        cudaFuncAttributes at;
        cudaError_t e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
        if (e == cudaSuccess) e = cudaDeviceGetAttribute(&smem, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev);
        if (e == cudaSuccess) e = cudaFuncGetAttributes(&at, (const void*)kernel);
        // the registers that the warps' shares add up to are there from the launch on: a share would be
        // waited for in vain otherwise
        if (e == cudaSuccess && (uint32_t)at.numRegs * kThreads < regs)
            return lrs_call_error(LRS_E_INTERNAL, "lrs_fp8_logits: %d registers a thread at launch", at.numRegs);
        if (e == cudaSuccess) smem -= (int)at.sharedSizeBytes;
        if (e == cudaSuccess) e = cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return lrs_call_error(LRS_E_CUDA, "lrs_fp8_logits: %s", cudaGetErrorString(e));
        info[dev].smem = smem;
        info[dev].sms = sms;
    }
    g.stages = ((uint32_t)info[dev].smem - 1024 - more) / g.stage_bytes;
    if (g.stages > kMaxStages) g.stages = kMaxStages;
    const uint32_t grid = g.tiles < (uint32_t)info[dev].sms ? g.tiles : (uint32_t)info[dev].sms;
    return launch_kernel("lrs_fp8_logits", kernel, grid, kThreads, g.stages * g.stage_bytes + 1024 + more, s, first, second, g);
}

template <typename T>
int run(const uint8_t* d_a, uint64_t ld_a, const uint8_t* d_w, uint64_t ld_w, uint32_t k, Args g, cudaStream_t s) {
    static DeviceInfo narrow_info[kMaxDevices], wide_info[kMaxDevices];
    g.wide_out = (uintptr_t)g.out % 16 == 0 && (g.rows == 1 || g.ld_out * sizeof(T) % 16 == 0);
    const bool narrow = g.rows <= (g.wide_out ? kNarrowAligned : kNarrowRows);
    g.tile_r = narrow ? (g.rows + 15) / 16 * 16 : kWideR;
    g.tile_v = narrow ? 128 : kWideV;
    g.row_tiles = (g.rows + g.tile_r - 1) / g.tile_r;
    const uint64_t tiles = (uint64_t)g.row_tiles * ((g.n + g.tile_v - 1) / g.tile_v);
    if (tiles > 0x7FFFFFFFu) return lrs_call_error(LRS_E_INVALID, "lrs_fp8_logits: rows x n too large");
    g.tiles = (uint32_t)tiles;
    g.first_bytes = 128 * kBlock;
    g.columns = narrow ? g.tile_r : g.tile_v;
    g.stage_bytes = g.first_bytes + g.columns * kBlock;
    g.buffers = 512 / g.columns < kMaxBuffers ? 512 / g.columns : kMaxBuffers;
    g.tmem_columns = 32;
    while (g.tmem_columns < g.buffers * g.columns) g.tmem_columns *= 2;
    CUtensorMap ma, mw;
    if (!code_map(&mw, d_w, g.n, k, ld_w, g.tile_v) || !code_map(&ma, d_a, g.rows, k, ld_a, g.tile_r))
        return lrs_call_error(LRS_E_INVALID, "lrs_fp8_logits: the codes cannot be mapped (ld too large?)");
    return narrow ? launch<T>(narrow_kernel<T>, narrow_info, mw, ma, g, 0, 0, s)
                  : launch<T>(wide_kernel<T>, wide_info, ma, mw, g, kWideRegs, kWideWarps * 32 * kPiece, s);
}

int logits(const uint8_t* d_a, uint64_t ld_a, const float* d_a_scale, uint64_t ld_as, const uint8_t* d_w, uint64_t ld_w,
           const float* d_w_scale, uint64_t ld_ws, uint32_t rows, uint32_t n, uint32_t k, void* d_out, int out_dtype,
           uint64_t ld_out, uint32_t copies, long long bound, void* stream) {
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
    g.copies = copies, g.bound = bound;
    const cudaStream_t s = (cudaStream_t)stream;
    return out_dtype == LRS_F32    ? run<float>(d_a, ld_a, d_w, ld_w, k, g, s)
           : out_dtype == LRS_BF16 ? run<__nv_bfloat16>(d_a, ld_a, d_w, ld_w, k, g, s)
                                   : run<__half>(d_a, ld_a, d_w, ld_w, k, g, s);
}

}  // namespace

extern "C" int lrs_fp8_logits(const uint8_t* d_a, uint64_t ld_a, const float* d_a_scale, uint64_t ld_as,
                              const uint8_t* d_w, uint64_t ld_w, const float* d_w_scale, uint64_t ld_ws, uint32_t rows,
                              uint32_t n, uint32_t k, void* d_out, int out_dtype, uint64_t ld_out, void* stream) {
    return logits(d_a, ld_a, d_a_scale, ld_as, d_w, ld_w, d_w_scale, ld_ws, rows, n, k, d_out, out_dtype, ld_out, ~0u,
                  kWaitCycles, stream);
}

extern "C" int lrs_test_fp8_logits_timeout(const uint8_t* d_a, uint64_t ld_a, const float* d_a_scale, uint64_t ld_as,
                                           const uint8_t* d_w, uint64_t ld_w, const float* d_w_scale, uint64_t ld_ws,
                                           uint32_t rows, uint32_t n, uint32_t k, void* d_out, int out_dtype,
                                           uint64_t ld_out, uint32_t steps, uint32_t bound_cycles, void* stream) {
    if (bound_cycles == 0) return lrs_call_error(LRS_E_INVALID, "lrs_test_fp8_logits_timeout: bound is 0");
    return logits(d_a, ld_a, d_a_scale, ld_as, d_w, ld_w, d_w_scale, ld_ws, rows, n, k, d_out, out_dtype, ld_out, steps,
                  bound_cycles, stream);
}
