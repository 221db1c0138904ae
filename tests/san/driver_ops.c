/* The operators around a fold (hg_ops.c) under -fsanitize=address,undefined with stubs.c's machine of one GPU: random and
 * boundary arguments for every entry point.  A call that succeeds has to reach stand-ins of the launches with a geometry
 * that covers the matrix, fits a grid and stays inside the workspace; a refused one none. */
#include <stdio.h>
#include <string.h>
#include "hcomm_gfx.h"
#include "hg_internal.h"
#include "hg_ops.h"

static unsigned long launches, bad, taken, refused, met[6];
static uint64_t state = 0x9E3779B97F4A7C15ull;
static uint64_t draw(void) { state ^= state << 13; state ^= state >> 7; state ^= state << 17; return state; }
static uint64_t below(uint64_t n) { return draw() % n; }

static void expect(int ok, const char* what)
{
    if (!ok) ++bad, fprintf(stderr, "wrong: %s\n", what);
}
static void grid(uint64_t wgs, uint64_t lanes) { ++launches; expect(wgs > 0 && wgs < (1ull << 31) && wgs * lanes < (1ull << 32), "grid"); }

static void mx_grid_ok(const HgMxGrid* g)
{
    grid(g->wgs, 256);
    expect(g->groups == (g->cols + 31) / 32 * 4 && (g->tile == 256 || g->tile == HG_MX_UNROLL * 256), "groups");
    if (g->rows_per_wg > 1) expect(g->rows_per_wg * g->groups <= g->tile && (uint64_t)g->wgs * g->rows_per_wg >= g->rows && g->tiles == 1, "rows of a workgroup");
    else expect((uint64_t)g->tiles * g->tile >= g->groups && (uint64_t)g->wgs == g->rows * g->tiles, "pieces of a row");
}
int hg_launch_mx_quantize(void* s, const void* a) { (void)s; ++met[0]; mx_grid_ok(&((const HgMxQuantize*)a)->grid); return 0; }
int hg_launch_mx_reduce(void* s, const void* a) { (void)s; ++met[1]; mx_grid_ok(&((const HgMxReduce*)a)->grid); return 0; }
int hg_launch_mx_product(void* s, const void* args)
{
    const HgMxProduct* p = (const HgMxProduct*)args;
    const uint64_t edge = p->form == HG_PRODUCT_DIRECT_16 ? 16 : p->form == HG_PRODUCT_DIRECT_32 || p->form == HG_PRODUCT_WAVE_32 ? 32 : p->form == HG_PRODUCT_MID_64 ? 64 : p->form == HG_PRODUCT_MID_128 ? 128 : 256;
    (void)s; ++met[2];
    grid(p->wgs, edge <= 32 ? 512 : 256);
    expect(p->wgs == (p->m + edge - 1) / edge * ((p->n + edge - 1) / edge), "tiles");
    return 0;
}
int hg_launch_norm(void* s, const void* args)
{
    const HgNorm* a = (const HgNorm*)args;
    (void)s; ++met[3];
    grid(a->wgs, a->span * a->rows_per_wg);
    expect(a->span * a->rows_per_wg <= 1024 && (uint64_t)a->span * a->vecs * 8 >= a->d.cols && (uint64_t)a->wgs * a->rows_per_wg >= a->d.rows, "norm");
    expect(a->span >= 64 ? a->span % 64 == 0 && (a->rows_per_wg == 1 || a->span <= 128) : a->span > 0 && a->span <= 32 && (a->span & (a->span - 1)) == 0, "span");
    return 0;
}
int hg_launch_norm_grad(void* s, const void* args)
{
    const HgNormGrad* a = (const HgNormGrad*)args;
    const uint64_t lanes = a->span < 64 ? 64 : a->span, rows = a->d.rows;
    (void)s; ++met[4];
    grid(a->chunks, lanes);
    expect(lanes <= 1024 && (uint64_t)a->span * a->vecs * 8 >= a->d.cols && a->pitch >= a->d.cols && a->pitch % 64 == 0 && (a->span < 64 || a->pitch <= a->span * a->vecs * 8), "lanes");
    expect(a->chunks * a->sums * a->pitch * 4 <= a->d.workspaceBytes, "workspace");
    if (a->by_gate) expect(a->chunks_per_gate * a->chunk_rows >= a->d.rowsPerGate && a->chunks == a->chunks_per_gate * a->gates && a->gates * a->d.rowsPerGate >= rows, "runs of a gate");
    else expect(a->chunks * a->chunk_rows >= rows && a->unit > 0 && (!a->d.dGate || (a->chunk_rows % a->d.rowsPerGate == 0 && a->unit == a->d.rowsPerGate)), "runs");
    expect(a->chunk_rows < (1ull << 32) && (uint64_t)a->unit * 64 + rows < (1ull << 32), "32 bits");
    return 0;
}
int hg_launch_norm_sums(void* s, const void* args)
{
    const HgNormGrad* a = (const HgNormGrad*)args;
    (void)s; ++met[5];
    grid(((a->d.cols + 63) / 64) * ((a->at_post >= 0) + (a->at_pre >= 0) + (a->at_gate >= 0 ? a->gates : 0)), 1024);
    expect(a->at_gate < 0 || a->gates + 2 < 65536, "sums");
    return 0;
}

static uint64_t size(uint64_t most)
{
    static const uint64_t edge[] = {0, 1, 2, 7, 8, 9, 31, 32, 33, 63, 64, 65, 255, 256, 257, 1023, 1024, 4096, 8192, 8193, 16384, 16385, 1ull << 20, 1ull << 24,
                                    (1ull << 31) - 1, 1ull << 31, 1ull << 32, 1ull << 34, (1ull << 34) + 1, 1ull << 48, 1ull << 63, ~0ull};
    switch (below(4)) {
        case 0: return edge[below(sizeof(edge) / sizeof(edge[0]))];
        case 1: return below(64);
        default: return below(1ull << (1 + below(most)));
    }
}
static uint64_t stride(uint64_t row) { return below(4) ? row + below(3) : size(30); }
static void* place(uint64_t slot) { return (void*)(uintptr_t)(below(60) ? (slot << 52) + 16 * below(2) + (below(8) ? 0 : 1 + below(15)) : (below(2) ? 0 : draw())); }
static HcommDataType type(void) { static const HcommDataType t[] = {HCOMM_DATA_TYPE_FP16, HCOMM_DATA_TYPE_BFP16, HCOMM_DATA_TYPE_FP32, HCOMM_DATA_TYPE_INT8}; return t[below(16) ? below(3) : 3]; }
static HcommGfxMxView view(uint64_t slot, uint64_t cols)
{
    const uint64_t nb = cols / 32 + (cols % 32 != 0), pad = below(2);
    HcommGfxMxView v = {place(slot), place(slot + 1), below(30) ? (nb + pad) * 16 : size(30), below(30) ? nb + pad : size(30)};
    if (below(8)) v.packed = (void*)((uintptr_t)v.packed / 16 * 16);
    return v;
}
static void done(int rc, unsigned long before)
{
    if (rc == HCCL_SUCCESS) ++taken;
    else ++refused, expect(launches == before, "a refused call launched");
}

int main(void)
{
    ThreadHandle th = 0;
    if (HcommThreadAllocWithStream(COMM_ENGINE_CPU_TS, (void*)(uintptr_t)0x5000, 0, &th)) return 2;
    for (int i = 0; i < 200000; ++i) {
        const uint64_t rows = size(24), cols = size(below(2) ? 12 : 26);
        const unsigned long before = launches;
        HcommGfxMxView a[HCOMM_GFX_MAX_RANKS], b[HCOMM_GFX_MAX_RANKS], out = view(1, cols);
        const uint32_t k = below(40) ? 1 + (uint32_t)below(below(8) ? 4 : HCOMM_GFX_MAX_RANKS) : (uint32_t)below(2) * 33;
        switch (below(5)) {
            case 0: done(HcommGfxMxQuantizeOnThread(th, &out, place(3), stride(cols), rows, cols, type()), before); break;
            case 1:
                for (uint32_t j = 0; j < HCOMM_GFX_MAX_RANKS; ++j) a[j] = view(10 + 2 * j, cols);
                done(HcommGfxMxReduceKOnThread(th, below(4) ? place(3) : NULL, stride(cols), type(), below(2) ? &out : NULL, a, k, below(2) ? place(5) : NULL, stride(cols), rows, cols), before);
                break;
            case 2: {
                const uint64_t n = size(24);
                for (uint32_t j = 0; j < HCOMM_GFX_MAX_RANKS; ++j) a[j] = view(10 + 2 * j, cols), b[j] = view(100 + 2 * j, cols);
                done(HcommGfxMxProductKOnThread(th, place(3), stride(n), type(), a, b, k, rows, n, cols), before);
                break;
            }
            case 3: {
                const void* srcs[HCOMM_GFX_MAX_RANKS];
                HcommGfxReduceNormDesc d;
                memset(&d, 0, sizeof(d));
                for (uint32_t j = 0; j < HCOMM_GFX_MAX_RANKS; ++j) srcs[j] = place(20 + j);
                d.rows = rows, d.cols = size(14), d.dataType = type(), d.paramType = below(2) ? d.dataType : HCOMM_DATA_TYPE_FP32, d.k = k, d.eps = 1e-5f;
                d.rowsPerGate = size(20), d.srcs = srcs, d.srcStride = stride(d.cols);
                d.residual = below(2) ? place(3) : NULL, d.residualStride = stride(d.cols), d.postWeight = below(2) ? place(4) : NULL, d.gate = below(2) ? place(6) : NULL;
                if (below(2)) d.preWeight = place(5), d.z = place(9);
                d.gateStride = stride(d.cols), d.sum = below(2) ? place(7) : NULL, d.sumStride = stride(d.cols), d.y = place(8), d.yStride = stride(d.cols), d.zStride = stride(d.cols);
                done(HcommGfxReduceNormOnThread(th, &d), before);
                break;
            }
            default: {
                HcommGfxReduceNormGradDesc d;
                uint64_t need = 0;
                memset(&d, 0, sizeof(d));
                d.rows = rows, d.cols = size(14), d.dataType = type(), d.paramType = below(2) ? d.dataType : HCOMM_DATA_TYPE_FP32, d.eps = 1e-5f, d.rowsPerGate = size(20);
                d.sum = place(3), d.sumStride = stride(d.cols), d.y = place(4), d.yStride = stride(d.cols), d.dy = place(5), d.dyStride = stride(d.cols);
                if (below(2)) d.preWeight = place(6), d.dz = place(7), d.dPreWeight = below(2) ? place(8) : NULL;
                if (below(2)) d.postWeight = place(9), d.dPostWeight = below(2) ? place(10) : NULL;
                if (below(2)) d.gate = place(11), d.dGate = below(2) ? place(12) : NULL;
                d.dzStride = stride(d.cols), d.gateStride = stride(d.cols), d.dGateStride = stride(d.cols), d.dSum = place(13), d.dSumStride = stride(d.cols);
                d.dResidual = below(2) ? place(14) : NULL, d.dResidualStride = stride(d.cols);
                const int rc = HcommGfxReduceNormGradWorkspaceBytes(&d, &need);
                d.workspace = (void*)(uintptr_t)(15ull << 52), d.workspaceBytes = rc ? size(30) : need - (need && !below(20));
                done(HcommGfxReduceNormGradOnThread(th, &d), before);
                break;
            }
        }
        HcommGfxLaunchLogClear(th);
    }
    HcommThreadFreeWithStream(&th, 1);
    for (int i = 0; i < 6; ++i) expect(met[i] > 1000, "an operator was hardly reached");
    printf("taken %lu refused %lu launches %lu bad %lu\n", taken, refused, launches, bad);
    return bad != 0;
}
