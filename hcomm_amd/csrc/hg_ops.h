/*
 * hg_ops.h - the operators around a fold: what the host code (hg_ops.c) hands to their launchers (hg_mx.hip,
 * hg_mx_product.hip, hg_norm.hip).  Plain C.  All geometry is decided on the host and checked there.
 */
#ifndef HG_OPS_H
#define HG_OPS_H

#include "hg_internal.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- microscaled 4-bit floating point --------------------------------------------------------------------- */

typedef struct {
    uint8_t* packed;
    uint8_t* scales;
    uint64_t packed_stride, scale_stride; /* bytes */
} HgMxView;

/*
 * Quantise and fold walk a matrix in groups of eight elements (a quarter of a block, one dword of elements), four
 * neighbouring lanes to a block.  A workgroup of 256 lanes takes a piece of `tile` groups of one row, or, where two rows or more
 * have that many groups together, `rows_per_wg` whole rows.  Host: every matrix that is one run of memory counts as one row.
 */
#define HG_MX_UNROLL 4u

typedef struct {
    uint64_t rows, cols;
    uint32_t groups;      /* of a row: 4 * ceil(cols / 32) */
    uint32_t tile;        /* groups to a workgroup: 256 or HG_MX_UNROLL * 256 */
    uint32_t tiles;       /* workgroups to a row */
    uint32_t rows_per_wg;
    uint32_t wgs;
} HgMxGrid;

typedef struct {
    HgMxGrid grid;
    HgMxView out;
    const void* src;
    uint64_t src_stride; /* elements */
    int dtype;
} HgMxQuantize;

typedef struct {
    HgMxGrid grid;
    HgMxView src[HCOMM_GFX_MAX_RANKS];
    HgMxView again; /* packed == NULL: not wanted */
    void* dst;      /* NULL: not wanted */
    const void* addend;
    uint64_t dst_stride, addend_stride; /* elements */
    uint32_t k;
    int dtype;
} HgMxReduce;

/* edge of a workgroup's results: 16, 32, 32 (one wavefront), 64, 128, 256 */
enum { HG_PRODUCT_DIRECT_16 = 0, HG_PRODUCT_DIRECT_32, HG_PRODUCT_WAVE_32, HG_PRODUCT_MID_64, HG_PRODUCT_MID_128, HG_PRODUCT_TILE };

typedef struct {
    HgMxView a[HCOMM_GFX_MAX_RANKS];
    HgMxView b[HCOMM_GFX_MAX_RANKS];
    void* dst;
    uint64_t dst_stride; /* elements */
    uint32_t m, n, cols, k;
    uint32_t form; /* HG_PRODUCT_* */
    uint32_t wgs;
    int dtype;
} HgMxProduct;

int hg_launch_mx_quantize(void* stream, const void* args); /* HgMxQuantize */
int hg_launch_mx_reduce(void* stream, const void* args);   /* HgMxReduce */
int hg_launch_mx_product(void* stream, const void* args);  /* HgMxProduct */

/* ---- norms behind a fold ------------------------------------------------------------------------------------ */

typedef struct {
    HcommGfxReduceNormDesc d; /* .srcs is not followed on the device: */
    const void* src[HCOMM_GFX_MAX_RANKS];
    uint32_t span;        /* lanes that share a row: 1 to 32, a power of two, or whole wavefronts */
    uint32_t vecs;        /* groups of eight elements a lane holds */
    uint32_t rows_per_wg;
    uint32_t wgs;
    uint32_t stream;      /* moves more than the L2s hold */
} HgNorm;

/*
 * The gradient walks the rows in `chunks` runs of `chunk_rows` rows, one workgroup a run, and joins the runs' sums in a
 * second launch.  by_gate: a run never crosses from one row of the gate to the next (`chunks_per_gate` runs to each), so
 * that the gate's gradient is joined from runs too, where there is more than one to a row of it; otherwise every run holds
 * whole gate rows and writes their gradients itself.
 */
typedef struct {
    HcommGfxReduceNormGradDesc d;
    uint64_t gates;           /* rows of the gate */
    uint64_t chunks, chunk_rows, chunks_per_gate;
    uint32_t by_gate;
    uint32_t span, vecs, stream;
    uint32_t unit;            /* rows that one set of lanes takes at a time where several share a wavefront */
    uint32_t sums;            /* rows of `pitch` fp32 a run writes to the workspace: post, pre, gate as wanted */
    uint32_t pitch;           /* cols rounded up to 64 */
    int at_post, at_pre, at_gate; /* which of them, -1: not there */
} HgNormGrad;

int hg_launch_norm(void* stream, const void* args);      /* HgNorm */
int hg_launch_norm_grad(void* stream, const void* args); /* HgNormGrad */
int hg_launch_norm_sums(void* stream, const void* args); /* HgNormGrad */

#ifdef __cplusplus
}
#endif
#endif
