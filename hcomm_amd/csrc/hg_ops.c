/*
 * hg_ops.c - the operators around a fold: argument checks, launch geometry, submission.  The kernels trust what is
 * checked here: strides that hold a row, ranges whose ends do not wrap, counts that fit the grid.
 */
#include <string.h>

#include "hg_host.h"
#include "hg_ops.h"

#define HG_LIMIT_LANES 0xffffffffull /* of a launch: the hardware counts them in 32 bits */
#define HG_LIMIT_ROWS 0x7fffffffull

static uint64_t elem_size(int dtype)
{
    return dtype == HCOMM_DATA_TYPE_FP32 ? 4u : (dtype == HCOMM_DATA_TYPE_FP16 || dtype == HCOMM_DATA_TYPE_BFP16) ? 2u : 0u;
}

/* ---- memory ranges ------------------------------------------------------------------------------------------ */

typedef struct {
    uintptr_t at;
    uint64_t bytes, row, stride; /* from its first byte to behind its last; of a row; from row to row */
} Range;

/* rows x row_bytes at `p`, `stride` bytes apart; 0 where a row does not fit its stride or the end wraps */
static int range_of(Range* r, const void* p, uint64_t rows, uint64_t row_bytes, uint64_t stride)
{
    uint64_t n;
    r->at = (uintptr_t)p;
    r->stride = stride;
    r->bytes = 0;
    r->row = row_bytes;
    if (rows == 0 || row_bytes == 0) return 1;
    if (rows > 1 && stride < row_bytes) return 0;
    if (rows == 1) r->stride = stride = row_bytes;
    if (__builtin_mul_overflow(rows - 1u, stride, &n) || __builtin_add_overflow(n, row_bytes, &n)) return 0;
    r->bytes = n;
    return !__builtin_add_overflow((uint64_t)r->at, n, &n);
}

static int dense_range(Range* r, const void* p, uint64_t rows, uint64_t cols, uint64_t stride, uint64_t es)
{
    uint64_t row, step;
    if ((uintptr_t)p % es != 0) return 0;
    if (__builtin_mul_overflow(cols, es, &row) || __builtin_mul_overflow(stride, es, &step)) return 0;
    if (rows == 1) step = row; /* a single row has no next one */
    return range_of(r, p, rows, row, step);
}

static int meets(const Range* a, const Range* b)
{
    if (!a->bytes || !b->bytes || a->at >= b->at + b->bytes || b->at >= a->at + a->bytes) return 0;
    if (a->stride != b->stride) return 1;
    /* two sets of columns of one larger matrix lie between one another without meeting */
    const uint64_t d = a->at <= b->at ? (b->at - a->at) % a->stride : (a->stride - (a->at - b->at) % a->stride) % a->stride;
    return d < a->row || d + b->row > a->stride;
}
static int same(const Range* a, const Range* b) { return a->at == b->at && a->bytes == b->bytes && a->stride == b->stride; }

/* an output may not meet any of these ranges, apart from the one that it may be itself */
static int clear_of(const Range* out, const Range* others, uint32_t n, const Range* may_be)
{
    for (uint32_t i = 0; i < n; ++i)
        if (&others[i] != out && meets(out, &others[i]) && !(&others[i] == may_be && same(out, may_be))) return 0;
    return 1;
}

/* ---- threads ------------------------------------------------------------------------------------------------- */

static int ready(const HgThread* t)
{
    if (hg_caller_is_batching()) return HCCL_E_NOT_SUPPORT;
    return hg_thread_free_for_caller(t);
}

static HcommGfxLaunchRecord record(uint32_t kind, int dtype, uint32_t op, uint32_t nseg, uint64_t bytes, uint64_t blocks, uint32_t rows)
{
    HcommGfxLaunchRecord r;
    memset(&r, 0, sizeof(r));
    r.kind = kind;
    r.dtype = (uint32_t)dtype;
    r.op = op;
    r.nseg = nseg;
    r.bytes = bytes;
    r.blocks = blocks;
    r.rows = rows;
    return r;
}

/* ---- microscaled 4-bit floating point --------------------------------------------------------------------------- */

#define HG_MX_MAX_COLS (1ull << 34)
#define HG_MX_PRODUCT_STRIDE (1ull << 23)

static uint64_t mx_blocks(uint64_t cols) { return cols / HCOMM_GFX_MX_BLOCK + (cols % HCOMM_GFX_MX_BLOCK != 0); }

static int mx_view(HgMxView* v, Range* packed, Range* scales, const HcommGfxMxView* in, uint64_t rows, uint64_t cols)
{
    const uint64_t blocks = mx_blocks(cols);
    v->packed = (uint8_t*)in->packed;
    v->scales = (uint8_t*)in->scales;
    v->packed_stride = rows > 1 ? in->packedStride : blocks * HCOMM_GFX_MX_BLOCK_BYTES; /* a single row has no next one */
    v->scale_stride = rows > 1 ? in->scaleStride : blocks;
    if ((uintptr_t)in->packed % HCOMM_GFX_MX_BLOCK_BYTES != 0) return 0;
    if (rows > 1 && in->packedStride % HCOMM_GFX_MX_BLOCK_BYTES != 0) return 0;
    return range_of(packed, in->packed, rows, blocks * HCOMM_GFX_MX_BLOCK_BYTES, in->packedStride) &&
           range_of(scales, in->scales, rows, blocks, in->scaleStride);
}

/*
 * A workgroup takes 256 groups, one to a lane, where that fills the GPU better: in every fold (dequantising 67.1M elements
 * 26.3 -> 24.9 us, 14.3M results of seven ranks 22.9 -> 22.3, 1,024 rows of 1,001 of eight ranks 7.5 -> 4.8) and in launches of up
 * to `few` workgroups of HG_MX_UNROLL groups a lane (1,024 x 1,001 quantised 8.5 -> 6.0).  Large quantisations keep several
 * groups in flight (67.1M elements 28.8 us; one group: 32.8).  Rows of up to half of that share a workgroup.
 */
#define HG_MX_FEW_WGS 1024u
#define HG_MX_ALWAYS 0xffffffffu

static int mx_grid(HgMxGrid* g, uint64_t rows, uint64_t cols, uint32_t few)
{
    uint32_t most = HG_MX_UNROLL * 256u;
    if (cols > HG_MX_MAX_COLS) return HCCL_E_NOT_SUPPORT;
    const uint64_t groups = mx_blocks(cols) * 4u;
    g->rows = rows;
    g->cols = cols;
    g->groups = (uint32_t)groups;
    const uint64_t in_row = (groups + most - 1u) / most, rows_of_wg = groups <= most / 2u ? most / groups : 1u;
    if (few == HG_MX_ALWAYS || rows / rows_of_wg <= few / in_row) most = 256u;
    g->tile = most;
    g->rows_per_wg = groups <= most / 2u && rows > 1 ? most / (uint32_t)groups : 1u;
    g->tiles = g->rows_per_wg > 1u ? 1u : (uint32_t)((groups + most - 1u) / most);
    const uint64_t wgs = rows / g->rows_per_wg + (rows % g->rows_per_wg != 0);
    if (wgs > HG_LIMIT_LANES / 256u / g->tiles) return HCCL_E_NOT_SUPPORT;
    g->wgs = (uint32_t)wgs * g->tiles;
    return HCCL_SUCCESS;
}

/* whether the rows follow one another without a gap, in whole blocks: then the matrix is one long row */
static int mx_is_run(const HgMxView* v, uint64_t cols)
{
    return cols % HCOMM_GFX_MX_BLOCK == 0 && v->scale_stride == cols / HCOMM_GFX_MX_BLOCK && v->packed_stride == cols / 2u;
}

int32_t HcommGfxMxQuantizeOnThread(
    ThreadHandle thread, const HcommGfxMxView* out, const void* src, uint64_t srcStride, uint64_t rows, uint64_t cols,
    HcommDataType srcType)
{
    if (!out || !out->packed || !out->scales || !src) return HCCL_E_PTR;
    HgThread* t = hg_thread_from_handle(thread);
    if (!t) return HCCL_E_PTR;
    const uint64_t es = elem_size((int)srcType);
    if (!es) return HCCL_E_PARA;
    HgMxQuantize a;
    memset(&a, 0, sizeof(a));
    int rc = cols > HG_MX_MAX_COLS ? HCCL_E_NOT_SUPPORT : HCCL_SUCCESS;
    if (rc == HCCL_SUCCESS) {
        Range r[3];
        if (!dense_range(&r[0], src, rows, cols, srcStride, es) || !mx_view(&a.out, &r[1], &r[2], out, rows, cols)) return HCCL_E_PARA;
        if (!clear_of(&r[1], r, 3, NULL) || !clear_of(&r[2], r, 3, NULL)) return HCCL_E_PARA;
        uint64_t all;
        const int run = rows > 1 && srcStride == cols && mx_is_run(&a.out, cols) && !__builtin_mul_overflow(rows, cols, &all) && all <= HG_MX_MAX_COLS;
        if (rows && cols) rc = run ? mx_grid(&a.grid, 1, all, HG_MX_FEW_WGS) : mx_grid(&a.grid, rows, cols, HG_MX_FEW_WGS);
    }
    if (rc == HCCL_SUCCESS) rc = ready(t);
    if (rc != HCCL_SUCCESS || rows == 0 || cols == 0) return rc;
    a.src = src;
    a.src_stride = rows > 1 ? srcStride : cols;
    a.dtype = (int)srcType;
    const HcommGfxLaunchRecord rec =
        record(HCOMM_GFX_KERNEL_MX_QUANTIZE, a.dtype, 255, 1, rows * mx_blocks(cols) * (HCOMM_GFX_MX_BLOCK_BYTES + 1u), a.grid.wgs, 0);
    return hg_submit_other(t, &rec, hg_launch_mx_quantize, &a);
}

int32_t HcommGfxMxReduceKOnThread(
    ThreadHandle thread, void* dst, uint64_t dstStride, HcommDataType dstType, const HcommGfxMxView* again,
    const HcommGfxMxView* srcs, uint32_t k, const void* addend, uint64_t addendStride, uint64_t rows, uint64_t cols)
{
    if (!dst && !again) return HCCL_E_PTR;
    if (again && (!again->packed || !again->scales)) return HCCL_E_PTR;
    if (!srcs) return HCCL_E_PTR;
    if (k == 0 || k > HCOMM_GFX_MAX_RANKS) return HCCL_E_PARA;
    for (uint32_t j = 0; j < k; ++j)
        if (!srcs[j].packed || !srcs[j].scales) return HCCL_E_PTR;
    HgThread* t = hg_thread_from_handle(thread);
    if (!t) return HCCL_E_PTR;
    const uint64_t es = elem_size((int)dstType);
    if (!es) return HCCL_E_PARA;
    HgMxReduce a;
    memset(&a, 0, sizeof(a));
    int rc = cols > HG_MX_MAX_COLS ? HCCL_E_NOT_SUPPORT : HCCL_SUCCESS;
    if (rc == HCCL_SUCCESS) {
        Range r[4 + 2 * HCOMM_GFX_MAX_RANKS]; /* dst, addend, again's two, the inputs' */
        memset(r, 0, sizeof(r));
        if (dst && !dense_range(&r[0], dst, rows, cols, dstStride, es)) return HCCL_E_PARA;
        if (addend && !dense_range(&r[1], addend, rows, cols, addendStride, es)) return HCCL_E_PARA;
        if (again && !mx_view(&a.again, &r[2], &r[3], again, rows, cols)) return HCCL_E_PARA;
        for (uint32_t j = 0; j < k; ++j)
            if (!mx_view(&a.src[j], &r[4 + 2 * j], &r[5 + 2 * j], &srcs[j], rows, cols)) return HCCL_E_PARA;
        if (!clear_of(&r[0], r, 4 + 2 * k, &r[1]) || !clear_of(&r[2], r, 4 + 2 * k, NULL) || !clear_of(&r[3], r, 4 + 2 * k, NULL))
            return HCCL_E_PARA;
        uint64_t all;
        int run = rows > 1 && (!dst || dstStride == cols) && (!addend || addendStride == cols) && (!again || mx_is_run(&a.again, cols)) &&
                  !__builtin_mul_overflow(rows, cols, &all) && all <= HG_MX_MAX_COLS;
        for (uint32_t j = 0; j < k && run; ++j) run = mx_is_run(&a.src[j], cols);
        if (rows && cols) rc = run ? mx_grid(&a.grid, 1, all, HG_MX_ALWAYS) : mx_grid(&a.grid, rows, cols, HG_MX_ALWAYS);
    }
    if (rc == HCCL_SUCCESS) rc = ready(t);
    if (rc != HCCL_SUCCESS || rows == 0 || cols == 0) return rc;
    a.dst = dst;
    a.dst_stride = rows > 1 ? dstStride : cols;
    a.addend = addend;
    a.addend_stride = rows > 1 ? addendStride : cols;
    a.k = k;
    a.dtype = (int)dstType;
    const uint64_t bytes = (dst ? rows * cols * es : 0) + (again ? rows * mx_blocks(cols) * (HCOMM_GFX_MX_BLOCK_BYTES + 1u) : 0);
    const HcommGfxLaunchRecord rec = record(HCOMM_GFX_KERNEL_MX_REDUCE, a.dtype, HCOMM_REDUCE_SUM, k, bytes, a.grid.wgs, 0);
    return hg_submit_other(t, &rec, hg_launch_mx_reduce, &a);
}

/* ---- product --------------------------------------------------------------------------------------------------------- */

/* what the forms through LDS ask for: a whole stage of columns (8 blocks), and ranks whose matrices have the same strides */
static int product_tiles(const HgMxProduct* a)
{
    if (mx_blocks(a->cols) < 8u) return 0;
    for (uint32_t j = 1; j < a->k; ++j)
        if (a->a[j].packed_stride != a->a[0].packed_stride || a->a[j].scale_stride != a->a[0].scale_stride ||
            a->b[j].packed_stride != a->b[0].packed_stride || a->b[j].scale_stride != a->b[0].scale_stride)
            return 0;
    return 1;
}

static uint64_t product_wgs(const HgMxProduct* a, uint32_t edge) { return (uint64_t)((a->m + edge - 1u) / edge) * ((a->n + edge - 1u) / edge); }

/*
 * The largest tiles of which there are enough for the CUs.  Measured, us for an inner length of 8,192 and n = 8,192 (edge 16 / 32 /
 * 64 / 128 / 256): m = 16: 12.3 / 11.3 / 12.4 / 23 / 47, m = 64: 33 / 21 / 13 / 23 / 47, m = 256: 121 / 76 / 25.5 / 25.1 / 50,
 * m = 512: 240 / 151 / 48 / 30 / 50, m = 1,024: 477 / 299 / 92 / 59 / 54, m = 4,096: 1,894 / 1,186 / 389 / 212 / 140; 200 x 200 x 512:
 * 2.7 / 3.1 / 3.5 / 4.8 / 10.4, 300 x 300 x 4,096: 7.1 / 6.8 / 7.3 / 14 / 32, 512 x 512 x 2,048: 7.4 / 5.0 / 5.4 / 8.5 / 18,
 * 33 x 8,000 x 2,048: 10.5 / 8.7 / 5.8 / 8.7 / 17, 300 x 1,200 x 4,096 with edge 32 / 64: 13.2 / 8.7.  Edge 32 has one workgroup to a
 * CU: up to 256 tiles of it run at once.
 * The rule counts tiles, not how full they are: more than 16,256 rows of b make enough tiles for edge 128, more than 32,512 for
 * 256, whatever m is.  Few rows of a lose by it (8 ranks' 1,024 columns, m = 1: n = 16,256 15.5 us, 16,384 24.3; n = 32,512 32.9, 32,768
 * 56.9; m = 64: 16.6 / 25.3, 35.0 / 59.6); the smaller edges have not been measured there.
 * Rows of fewer than 16 blocks: a wavefront for every 32 x 32 results instead of eight that share so little, from about as many
 * tiles on as a wavefront takes fours of blocks (8 wavefronts / 1 / edge 64 / 128): 1,024 x 1,024 results of one rank's 32 columns
 * 6.7 / 3.4, of four ranks' 165 8.3 / 5.6, of 16 ranks' 30 9.6 / 8.3; 512 x 512 of 8 ranks' 32 3.3 / 4.8; 4,096 x 8,192 of one rank's 32
 * 153 / 28; 410 x 3,924 of one rank's 250 12.5 / 5.8 / 7.2 / 6.7, of four ranks' 250 18.7 / 12.8 / 11.7 / 9.3.
 */
static int product_form(HgMxProduct* a)
{
    const uint64_t blocks = mx_blocks(a->cols), fours = a->k * ((blocks + 3u) / 4u), of_32 = product_wgs(a, 32u);
    const int tiles = product_tiles(a);
    uint32_t edge = 16u;
    a->form = HG_PRODUCT_DIRECT_16;
    if (tiles && product_wgs(a, 256u) >= 128u) {
        edge = 256u;
        a->form = HG_PRODUCT_TILE;
    } else if (blocks < 16u && (!tiles || fours <= 2u) && of_32 >= (fours < 13u ? 192u + 64u * fours : 1024u)) {
        edge = 32u;
        a->form = HG_PRODUCT_WAVE_32;
    } else if (tiles && product_wgs(a, 128u) >= 128u) {
        edge = 128u;
        a->form = HG_PRODUCT_MID_128;
    } else if (tiles && a->m > 32u && a->n > 32u && of_32 > 256u) {
        edge = 64u;
        a->form = HG_PRODUCT_MID_64;
    } else if (a->m > 16u && a->n > 16u && of_32 >= 64u) {
        edge = 32u;
        a->form = HG_PRODUCT_DIRECT_32;
    }
    a->wgs = (uint32_t)product_wgs(a, edge);
    return product_wgs(a, edge) <= HG_LIMIT_LANES / 512u; /* the direct forms' workgroups */
}

int32_t HcommGfxMxProductKOnThread(
    ThreadHandle thread, void* dst, uint64_t dstStride, HcommDataType dstType, const HcommGfxMxView* a,
    const HcommGfxMxView* b, uint32_t k, uint64_t m, uint64_t n, uint64_t cols)
{
    if (!dst || !a || !b) return HCCL_E_PTR;
    if (k == 0 || k > HCOMM_GFX_MAX_RANKS) return HCCL_E_PARA;
    for (uint32_t j = 0; j < k; ++j)
        if (!a[j].packed || !a[j].scales || !b[j].packed || !b[j].scales) return HCCL_E_PTR;
    HgThread* t = hg_thread_from_handle(thread);
    if (!t) return HCCL_E_PTR;
    const uint64_t es = elem_size((int)dstType);
    if (!es || cols == 0) return HCCL_E_PARA;
    HgMxProduct p;
    memset(&p, 0, sizeof(p));
    const int large = m > HG_LIMIT_ROWS - 512u || n > HG_LIMIT_ROWS - 512u || mx_blocks(cols) * HCOMM_GFX_MX_BLOCK_BYTES >= HG_MX_PRODUCT_STRIDE;
    int rc = large ? HCCL_E_NOT_SUPPORT : HCCL_SUCCESS;
    if (rc == HCCL_SUCCESS) {
        Range r[1 + 4 * HCOMM_GFX_MAX_RANKS];
        memset(r, 0, sizeof(r));
        if (!dense_range(&r[0], dst, m, n, dstStride, es)) return HCCL_E_PARA;
        for (uint32_t j = 0; j < k; ++j) {
            if (!mx_view(&p.a[j], &r[1 + 4 * j], &r[2 + 4 * j], &a[j], m, cols)) return HCCL_E_PARA;
            if (!mx_view(&p.b[j], &r[3 + 4 * j], &r[4 + 4 * j], &b[j], n, cols)) return HCCL_E_PARA;
            /* 256 rows of a tile are told apart by 32-bit offsets */
            if (m > 1 && (a[j].packedStride >= HG_MX_PRODUCT_STRIDE || a[j].scaleStride >= HG_MX_PRODUCT_STRIDE)) rc = HCCL_E_NOT_SUPPORT;
            if (n > 1 && (b[j].packedStride >= HG_MX_PRODUCT_STRIDE || b[j].scaleStride >= HG_MX_PRODUCT_STRIDE)) rc = HCCL_E_NOT_SUPPORT;
        }
        if (!clear_of(&r[0], r, 1 + 4 * k, NULL)) return HCCL_E_PARA;
        p.m = (uint32_t)m;
        p.n = (uint32_t)n;
        p.cols = (uint32_t)cols;
        p.k = k;
        if (rc == HCCL_SUCCESS && !product_form(&p)) rc = HCCL_E_NOT_SUPPORT;
    }
    if (rc == HCCL_SUCCESS) rc = ready(t);
    if (rc != HCCL_SUCCESS || m == 0 || n == 0) return rc;
    p.dst = dst;
    p.dst_stride = m > 1 ? dstStride : n;
    p.dtype = (int)dstType;
    const HcommGfxLaunchRecord rec = record(HCOMM_GFX_KERNEL_MX_PRODUCT, p.dtype, HCOMM_REDUCE_SUM, k, m * n * es, p.wgs, p.form);
    return hg_submit_other(t, &rec, hg_launch_mx_product, &p);
}

/* ---- norms behind a fold ------------------------------------------------------------------------------------------------ */

/* Lanes to a row of `cols` with `vecs` groups of eight elements each: 1 to 32 of a wavefront, or whole wavefronts. */
static uint32_t row_span(uint64_t cols, uint32_t vecs)
{
    const uint32_t lanes = (uint32_t)((cols + 8u * vecs - 1u) / (8u * vecs));
    for (uint32_t s = 1; s <= 32u; s *= 2u)
        if (lanes <= s) return s;
    return (lanes + 63u) / 64u * 64u;
}

#define HG_L2_BYTES (32ull << 20) /* of the eight XCDs together */

static int norm_types(HcommDataType data, HcommDataType param)
{
    return elem_size((int)data) != 0 && (param == data || param == HCOMM_DATA_TYPE_FP32);
}

/* eps >= 0 and neither number NaN or infinite */
static int norm_numbers(float scale, float eps) { return eps >= 0.0f && eps - eps == 0.0f && scale - scale == 0.0f; }

static uint64_t gate_rows(uint64_t rows, uint64_t per) { return rows / per + (rows % per != 0); }

int32_t HcommGfxReduceNormOnThread(ThreadHandle thread, const HcommGfxReduceNormDesc* desc)
{
    if (!desc || !desc->srcs || !desc->y) return HCCL_E_PTR;
    if (!desc->preWeight != !desc->z) return HCCL_E_PTR;
    if (desc->k == 0 || desc->k > HCOMM_GFX_MAX_RANKS) return HCCL_E_PARA;
    for (uint32_t j = 0; j < desc->k; ++j)
        if (!desc->srcs[j]) return HCCL_E_PTR;
    HgThread* t = hg_thread_from_handle(thread);
    if (!t) return HCCL_E_PTR;
    if (!norm_types(desc->dataType, desc->paramType) || !norm_numbers(desc->residualScale, desc->eps)) return HCCL_E_PARA;
    if (desc->gate && desc->rowsPerGate == 0) return HCCL_E_PARA;
    HgNorm a;
    memset(&a, 0, sizeof(a));
    a.d = *desc;
    const uint64_t rows = desc->rows, cols = desc->cols, es = elem_size((int)desc->dataType), ps = elem_size((int)desc->paramType);
    int rc = cols > HCOMM_GFX_NORM_MAX_COLS || rows > HG_LIMIT_ROWS ? HCCL_E_NOT_SUPPORT : HCCL_SUCCESS;
    if (rc == HCCL_SUCCESS) {
        enum { SUM, Y, Z, RES, POST, PRE, GATE, SRC };
        Range r[SRC + HCOMM_GFX_MAX_RANKS];
        memset(r, 0, sizeof(r));
        if (desc->sum && !dense_range(&r[SUM], desc->sum, rows, cols, desc->sumStride, es)) return HCCL_E_PARA;
        if (!dense_range(&r[Y], desc->y, rows, cols, desc->yStride, es)) return HCCL_E_PARA;
        if (desc->z && !dense_range(&r[Z], desc->z, rows, cols, desc->zStride, es)) return HCCL_E_PARA;
        if (desc->residual && !dense_range(&r[RES], desc->residual, rows, cols, desc->residualStride, es)) return HCCL_E_PARA;
        if (desc->postWeight && !dense_range(&r[POST], desc->postWeight, 1, cols, cols, ps)) return HCCL_E_PARA;
        if (desc->preWeight && !dense_range(&r[PRE], desc->preWeight, 1, cols, cols, ps)) return HCCL_E_PARA;
        if (desc->gate && !dense_range(&r[GATE], desc->gate, gate_rows(rows, desc->rowsPerGate), cols, desc->gateStride, ps)) return HCCL_E_PARA;
        for (uint32_t j = 0; j < desc->k; ++j)
            if (!dense_range(&r[SRC + j], desc->srcs[j], rows, cols, desc->srcStride, es)) return HCCL_E_PARA;
        const uint32_t n = SRC + desc->k;
        if (!clear_of(&r[SUM], r, n, &r[SRC]) || !clear_of(&r[Y], r, n, &r[RES]) || !clear_of(&r[Z], r, n, NULL)) return HCCL_E_PARA;
        /*
         * One group of eight to a lane as far as 1024 lanes reach: two in half the lanes take longer where rows are few (one row of
         * 8,192 bf16, 4 partials: 6.2 us against 5.2) and about as long where they are many (5,461 x 6,144: 119 against 98;
         * 4,096 x 8,192: 108 against 118).  Rows of up to 256 share a wavefront: 524,288 x 64 took 349 us with one each, 93 so.
         */
        a.vecs = cols > 8192u ? 2u : 1u;
        a.span = row_span(cols, a.vecs);
        a.rows_per_wg = a.span <= 128u && a.vecs == 1u ? 256u / a.span : 1u;
        a.wgs = (uint32_t)((rows + a.rows_per_wg - 1u) / a.rows_per_wg);
        if (a.wgs > HG_LIMIT_LANES / (a.span * a.rows_per_wg)) rc = HCCL_E_NOT_SUPPORT;
    }
    if (rc == HCCL_SUCCESS) rc = ready(t);
    if (rc != HCCL_SUCCESS || rows == 0 || cols == 0) return rc;
    for (uint32_t j = 0; j < desc->k; ++j) a.src[j] = desc->srcs[j];
    a.d.srcs = NULL;
    if (!a.d.gate || a.d.rowsPerGate > rows) a.d.rowsPerGate = rows;
    const uint64_t bytes = rows * cols * es * (1u + (desc->sum != NULL) + (desc->z != NULL));
    a.stream = bytes + rows * cols * es * desc->k > HG_L2_BYTES;
    const HcommGfxLaunchRecord rec = record(HCOMM_GFX_KERNEL_NORM, (int)desc->dataType, HCOMM_REDUCE_SUM, desc->k, bytes, a.wgs, a.span);
    return hg_submit_other(t, &rec, hg_launch_norm, &a);
}

/*
 * Runs of rows: as many as run at once, with up to 8 wavefronts to each of the CUs (their registers allow no more).  Enough to
 * keep every CU loading, few enough that the runs' sums stay a small part of the traffic; a few more than that would have the
 * card wait for a second turn (5,461 x 6,144 bf16: 341 runs of 6 wavefronts 129 us).
 * With the gate's gradient a run ends with a row of the gate, so that numbers of gate rows just above half or all of these runs
 * leave CUs without one: gates of 128 rows x 4,096 take 1.21 us each where there are 192 or 256, 1.55 where 129, 1.49 where 257.
 */
#define HG_NORM_GRAD_CUS 256u
#define HG_NORM_GRAD_WAVES 8u

/* the geometry, from the sizes and from which parameters' gradients are wanted alone */
static void norm_grad_shape(HgNormGrad* a)
{
    HcommGfxReduceNormGradDesc* d = &a->d;
    const uint64_t rows = d->rows;
    a->vecs = d->cols > 4096u ? 2u : 1u;
    a->span = row_span(d->cols, a->vecs);
    const uint32_t waves = a->span < 64u ? 1u : a->span / 64u;
    const uint64_t most = HG_NORM_GRAD_CUS * (waves > HG_NORM_GRAD_WAVES ? 1u : HG_NORM_GRAD_WAVES / waves);
    const uint64_t sets = a->span < 64u ? 64u / a->span : 1u; /* of lanes to a wavefront, a row each */
    if (!d->gate || d->rowsPerGate > rows) d->rowsPerGate = rows ? rows : 1u;
    a->gates = d->gate ? gate_rows(rows, d->rowsPerGate) : 0u;
    const int gate_wanted = d->gate && d->dGate;
    a->by_gate = gate_wanted && a->gates < most;
    a->chunks = a->chunk_rows = a->chunks_per_gate = 0;
    a->unit = 1;
    if (rows && a->by_gate) {
        uint64_t per = most / a->gates;
        if (per > d->rowsPerGate) per = d->rowsPerGate;
        /* a few rows one after another take less than the join of many rows of the gate: 900 x 1,024 with a row for every 2: 30.0 -> 12.9
           us, 2,000 x 1,024 for every 8: 24.6 -> 18.3 */
        if (d->rowsPerGate <= 8u && a->gates * ((d->cols + 63u) / 64u) > 1024u) per = 1u;
        a->chunk_rows = (d->rowsPerGate + per - 1u) / per;
        if (a->chunk_rows < sets) a->chunk_rows = sets;
        a->chunks_per_gate = (d->rowsPerGate + a->chunk_rows - 1u) / a->chunk_rows;
        a->chunks = a->chunks_per_gate * a->gates;
    } else if (rows) {
        /* with a gradient of the gate to write, whole gate rows */
        const uint64_t unit = gate_wanted ? d->rowsPerGate : 1u, units = gate_rows(rows, unit);
        a->unit = (uint32_t)unit;
        const uint64_t each = (units + most - 1u) / most;
        a->chunk_rows = (each < sets ? sets : each) * unit;
        a->chunks = gate_rows(rows, a->chunk_rows);
    }
    a->sums = 0;
    a->pitch = (uint32_t)(d->cols + 63u) / 64u * 64u;
    a->at_post = d->dPostWeight ? (int)a->sums++ : -1;
    a->at_pre = d->dPreWeight ? (int)a->sums++ : -1;
    a->at_gate = a->by_gate && a->chunks_per_gate > 1u ? (int)a->sums++ : -1; /* 536 x 626 with a row for each: 23.9 us joined, 10.8 not */
}

static uint64_t norm_grad_workspace(const HgNormGrad* a) { return a->chunks * a->sums * a->pitch * sizeof(float); }

int32_t HcommGfxReduceNormGradWorkspaceBytes(const HcommGfxReduceNormGradDesc* desc, uint64_t* bytes)
{
    if (!desc || !bytes) return HCCL_E_PTR;
    if (desc->gate && desc->rowsPerGate == 0) return HCCL_E_PARA;
    if (desc->cols > HCOMM_GFX_NORM_MAX_COLS || desc->rows > HG_LIMIT_ROWS) return HCCL_E_NOT_SUPPORT;
    HgNormGrad a;
    memset(&a, 0, sizeof(a));
    a.d = *desc;
    if (desc->cols) norm_grad_shape(&a);
    *bytes = norm_grad_workspace(&a);
    return HCCL_SUCCESS;
}

int32_t HcommGfxReduceNormGradOnThread(ThreadHandle thread, const HcommGfxReduceNormGradDesc* desc)
{
    if (!desc || !desc->sum || !desc->dy || !desc->dSum) return HCCL_E_PTR;
    if (!desc->preWeight != !desc->dz || (desc->preWeight && !desc->y)) return HCCL_E_PTR;
    HgThread* t = hg_thread_from_handle(thread);
    if (!t) return HCCL_E_PTR;
    if (!norm_types(desc->dataType, desc->paramType) || !norm_numbers(desc->residualScale, desc->eps)) return HCCL_E_PARA;
    if (desc->gate && desc->rowsPerGate == 0) return HCCL_E_PARA;
    if ((desc->dPostWeight && !desc->postWeight) || (desc->dPreWeight && !desc->preWeight) || (desc->dGate && !desc->gate)) return HCCL_E_PARA;
    HgNormGrad a;
    memset(&a, 0, sizeof(a));
    a.d = *desc;
    const uint64_t rows = desc->rows, cols = desc->cols, es = elem_size((int)desc->dataType), ps = elem_size((int)desc->paramType);
    int rc = cols > HCOMM_GFX_NORM_MAX_COLS || rows > HG_LIMIT_ROWS ? HCCL_E_NOT_SUPPORT : HCCL_SUCCESS;
    if (rc == HCCL_SUCCESS) {
        if (cols) norm_grad_shape(&a);
        const uint64_t need = norm_grad_workspace(&a), gates = desc->gate ? gate_rows(rows, desc->rowsPerGate) : 0u;
        if (need && !desc->workspace) return HCCL_E_PTR;
        if (need && (desc->workspaceBytes < need || (uintptr_t)desc->workspace % 16u != 0)) return HCCL_E_PARA;
        enum { DSUM, DRES, DPOST, DPRE, DGATE, WORK, OUTPUTS, SUM = OUTPUTS, Y, DY, DZ, POST, PRE, GATE, ALL };
        Range r[ALL];
        memset(r, 0, sizeof(r));
        int ok = dense_range(&r[DSUM], desc->dSum, rows, cols, desc->dSumStride, es) && dense_range(&r[SUM], desc->sum, rows, cols, desc->sumStride, es) &&
                 dense_range(&r[DY], desc->dy, rows, cols, desc->dyStride, es);
        if (ok && desc->dResidual) ok = dense_range(&r[DRES], desc->dResidual, rows, cols, desc->dResidualStride, es);
        if (ok && desc->preWeight)
            ok = dense_range(&r[Y], desc->y, rows, cols, desc->yStride, es) && dense_range(&r[DZ], desc->dz, rows, cols, desc->dzStride, es) &&
                 dense_range(&r[PRE], desc->preWeight, 1, cols, cols, ps);
        if (ok && desc->postWeight) ok = dense_range(&r[POST], desc->postWeight, 1, cols, cols, ps);
        if (ok && desc->gate) ok = dense_range(&r[GATE], desc->gate, gates, cols, desc->gateStride, ps);
        if (ok && desc->dPostWeight) ok = dense_range(&r[DPOST], desc->dPostWeight, 1, cols, cols, ps);
        if (ok && desc->dPreWeight) ok = dense_range(&r[DPRE], desc->dPreWeight, 1, cols, cols, ps);
        if (ok && desc->dGate) ok = dense_range(&r[DGATE], desc->dGate, gates, cols, desc->dGateStride, ps);
        if (ok && need) ok = range_of(&r[WORK], desc->workspace, 1, need, need);
        if (!ok) return HCCL_E_PARA;
        for (uint32_t o = 0; o < OUTPUTS; ++o) {
            /* the gradient of a matrix may overwrite the matrix, and either of the two dy - but not both */
            const Range* may = NULL;
            if (o == DSUM) may = same(&r[DSUM], &r[SUM]) ? &r[SUM] : &r[DY];
            if (o == DRES) may = same(&r[DRES], &r[Y]) ? &r[Y] : &r[DY];
            if (!clear_of(&r[o], r, ALL, may)) return HCCL_E_PARA;
        }
    }
    if (rc == HCCL_SUCCESS) rc = ready(t);
    if (rc != HCCL_SUCCESS || cols == 0) return rc;
    a.stream = rows * cols * es * 4u > HG_L2_BYTES; /* sum, dy and what is written, at least */
    if (a.chunks) {
        const HcommGfxLaunchRecord rec = record(
            HCOMM_GFX_KERNEL_NORM_GRAD, (int)desc->dataType, 255, 1, rows * cols * es * (1u + (desc->dResidual != NULL)), a.chunks, a.span);
        rc = hg_submit_other(t, &rec, hg_launch_norm_grad, &a);
    }
    if (rc == HCCL_SUCCESS && a.sums) {
        const uint64_t results = (a.at_post >= 0) + (a.at_pre >= 0) + (a.at_gate >= 0 ? a.gates : 0u);
        if (results) {
            const HcommGfxLaunchRecord rec = record(HCOMM_GFX_KERNEL_NORM_SUMS, (int)desc->paramType, HCOMM_REDUCE_SUM, (uint32_t)a.chunks,
                                                    results * cols * ps, results * ((cols + 63u) / 64u), 0);
            rc = hg_submit_other(t, &rec, hg_launch_norm_sums, &a);
        }
    }
    return rc;
}
