/* rust_ops_abi.c — the ABI that rust/src/ops.rs declares, checked against the C header and the built
 * library without a GPU: each `extern "C"` function as a function-pointer type written from the Rust
 * signature must be the header's, and every symbol must be in the library. */
#include <dlfcn.h>
#include <stddef.h>
#include <stdint.h>
#include <stdio.h>

#include "../../include/llamars_sampler.h"

_Static_assert(sizeof(lrs_draw_params) == 16, "lrs_draw_params size");
_Static_assert(offsetof(lrs_draw_params, temperature) == 0, "temperature");
_Static_assert(offsetof(lrs_draw_params, top_k) == 4, "top_k");
_Static_assert(offsetof(lrs_draw_params, top_p) == 8, "top_p");
_Static_assert(offsetof(lrs_draw_params, min_p) == 12, "min_p");
_Static_assert(LRS_F32 == 0 && LRS_BF16 == 1 && LRS_F16 == 2, "element types");

typedef int (*rs_lrs_draw_device)(const void *, int, uint32_t, uint32_t, uint64_t, const lrs_draw_params *, const float *,
                                  uint32_t *, float *, uint32_t *, int32_t *, void *);
typedef int (*rs_lrs_quantize_rows)(const void *, int, uint32_t, uint32_t, uint64_t, uint8_t *, uint64_t, float *,
                                    uint64_t, void *);
typedef int (*rs_lrs_quantize_blocks)(const void *, int, uint32_t, uint32_t, uint64_t, uint8_t *, uint64_t, float *,
                                      uint64_t, void *);
typedef int (*rs_lrs_fp8_logits)(const uint8_t *, uint64_t, const float *, uint64_t, const uint8_t *, uint64_t,
                                 const float *, uint64_t, uint32_t, uint32_t, uint32_t, void *, int, uint64_t, void *);

#define SAME(f) _Static_assert(__builtin_types_compatible_p(__typeof__(&f), rs_##f), #f " differs from ops.rs")
SAME(lrs_draw_device);
SAME(lrs_quantize_rows);
SAME(lrs_quantize_blocks);
SAME(lrs_fp8_logits);

int main(int argc, char **argv) {
    void *h = argc > 1 ? dlopen(argv[1], RTLD_NOW | RTLD_LOCAL) : NULL;
    if (!h) return 2;
    const rs_lrs_draw_device draw = (rs_lrs_draw_device)dlsym(h, "lrs_draw_device");
    const rs_lrs_quantize_rows rows = (rs_lrs_quantize_rows)dlsym(h, "lrs_quantize_rows");
    const rs_lrs_quantize_blocks blocks = (rs_lrs_quantize_blocks)dlsym(h, "lrs_quantize_blocks");
    const rs_lrs_fp8_logits logits = (rs_lrs_fp8_logits)dlsym(h, "lrs_fp8_logits");
    if (!draw || !rows || !blocks || !logits) return 3;
    /* no rows: nothing to do; null buffers: refused before any device work */
    if (draw(NULL, 0, 0, 0, 0, NULL, NULL, NULL, NULL, NULL, NULL, NULL) != LRS_OK) return 4;
    if (draw(NULL, 0, 1, 8, 8, NULL, NULL, NULL, NULL, NULL, NULL, NULL) != LRS_E_INVALID) return 5;
    if (rows(NULL, 0, 1, 8, 8, NULL, 8, NULL, 1, NULL) != LRS_E_INVALID) return 6;
    if (blocks(NULL, 0, 1, 8, 8, NULL, 8, NULL, 1, NULL) != LRS_E_INVALID) return 7;
    if (logits(NULL, 16, NULL, 1, NULL, 16, NULL, 1, 1, 1, 16, NULL, 0, 1, NULL) != LRS_E_INVALID) return 8;
    printf("rust ops ABI ok\n");
    return 0;
}
